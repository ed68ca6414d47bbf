"""Generates the raw Rust binding of include/tract_rocm.h.

Usage: ``python include/gen_rust_ffi.py`` prints the `extern "C"` block; ``python include/gen_rust_ffi.py --write``
rewrites rust/tract-rocm/src/ffi.rs (opaque handles, enum constants, the block and the KO -> error helper).
tests/test_abi_cpu.py checks that the committed ffi.rs is this script's output for today's header, and that every
`ffi::trocm_*` call in the Rust sources names a declared entry point with the declared number of arguments.
"""
from __future__ import annotations

import os
import re

HERE = os.path.dirname(os.path.abspath(__file__))

SCALARS = {"int": "c_int", "int64_t": "i64", "size_t": "usize", "float": "f32", "uint64_t": "u64", "int32_t": "i32", "unsigned": "c_uint",
           "void": "c_void", "char": "c_char"}
RUST_KEYWORDS = {"type", "ref", "in", "move", "match", "loop", "mod", "fn", "use", "box"}


def declarations(header_text: str):
    """[(name, return C type, [(C type, parameter name), ...])] in header order."""
    text = re.sub(r"/\*.*?\*/", "", header_text, flags=re.S)
    text = re.sub(r"^\s*#.*$", "", text, flags=re.M)
    out = []
    for m in re.finditer(r"([A-Za-z_][A-Za-z0-9_ \*]*?)\b(trocm_[a-z0-9_]+)\s*\(([^;{}]*?)\)\s*;", text, flags=re.S):
        ret, name, params = m.group(1).strip(), m.group(2), " ".join(m.group(3).split())
        if ret.startswith("typedef"):
            continue
        plist = []
        if params and params != "void":
            for prm in params.split(","):
                prm = prm.strip()
                pm = re.match(r"^(.*?)([A-Za-z_][A-Za-z0-9_]*)$", prm)
                plist.append((pm.group(1).strip(), pm.group(2)))
        out.append((name, ret, plist))
    return out


def rust_type(ctype: str) -> str:
    """C parameter type -> Rust FFI type: `const T *const *` reads right to left."""
    toks = re.findall(r"\*|const|[A-Za-z_][A-Za-z0-9_]*", ctype)
    base = [t for t in toks if t not in ("*", "const")]
    assert len(base) == 1, ctype
    assert base[0] in SCALARS or base[0].startswith("trocm_"), f"no Rust type is known for {ctype}"
    rust = SCALARS.get(base[0], base[0])   # opaque structs keep their names
    stars = [i for i, t in enumerate(toks) if t == "*"]
    if not stars:
        return rust
    # constness of the pointee at each level: a `const` directly before the base or directly after a star
    pointee_const = "const" in toks[:stars[0]]
    for idx, si in enumerate(stars):
        rust = ("*const " if pointee_const else "*mut ") + rust
        nxt = stars[idx + 1] if idx + 1 < len(stars) else len(toks)
        pointee_const = "const" in toks[si + 1:nxt]
    return rust


def rust_block(header_text: str) -> str:
    lines = ['extern "C" {']
    for name, ret, params in declarations(header_text):
        args = ", ".join(f"{(p + '_') if p in RUST_KEYWORDS else p}: {rust_type(t)}" for t, p in params)
        r = rust_type(ret)
        lines.append(f"    pub fn {name}({args}) -> {r};")
    lines.append("}")
    return "\n".join(lines)


def enum_constants(header_text: str):
    """[(NAME, value)] of every enumerator of the header's enums, in order."""
    text = re.sub(r"/\*.*?\*/", "", header_text, flags=re.S)
    out = []
    for body in re.findall(r"enum\s*[A-Za-z_0-9]*\s*\{(.*?)\}", text, flags=re.S):
        nxt = 0
        for item in body.split(","):
            item = item.strip()
            if not item:
                continue
            m = re.match(r"^([A-Z][A-Z0-9_]*)\s*(?:=\s*(-?\d+))?$", item)
            assert m, item
            val = int(m.group(2)) if m.group(2) is not None else nxt
            out.append((m.group(1), val))
            nxt = val + 1
    return out


def opaque_types(header_text: str):
    return sorted(set(re.findall(r"typedef\s+struct\s+(trocm_[a-z0-9_]+)\s+\1\s*;", header_text)))


def rust_file(header_text: str) -> str:
    """The whole of rust/tract-rocm/src/ffi.rs."""
    lines = ["// Raw binding of include/tract_rocm.h.  GENERATED by include/gen_rust_ffi.py --write: do not edit by hand.",
             "// Error convention (the reverse of api/ffi/src/lib.rs:18-62): every call returns 0 = OK or 1 = KO, and the",
             "// message of the last KO on the calling thread is read with trocm_last_error().",
             "#![allow(non_camel_case_types, clippy::too_many_arguments)]",
             "use std::os::raw::{c_char, c_int, c_void};",
             ""]
    for t in opaque_types(header_text):
        lines += ["#[repr(C)]", f"pub struct {t} {{", "    _private: [u8; 0],", "}"]
    lines.append("")
    for name, val in enum_constants(header_text):
        lines.append(f"pub const {name}: c_int = {val};")
    lines += ["", rust_block(header_text), "",
              "/// KO -> an error that carries the library's message.",
              "pub fn check(rc: c_int) -> tract_core::internal::TractResult<()> {",
              "    if rc == 0 {",
              "        return Ok(());",
              "    }",
              "    let msg = unsafe { std::ffi::CStr::from_ptr(trocm_last_error()) }.to_string_lossy().into_owned();",
              "    tract_core::internal::bail!(\"tract-rocm: {msg}\")",
              "}",
              ""]
    return "\n".join(lines)


FFI_RS = os.path.join(HERE, "..", "rust", "tract-rocm", "src", "ffi.rs")

if __name__ == "__main__":
    import sys
    header = open(os.path.join(HERE, "tract_rocm.h")).read()
    if "--write" in sys.argv:
        with open(FFI_RS, "w") as f:
            f.write(rust_file(header))
        print("wrote", os.path.normpath(FFI_RS))
    else:
        print(rust_block(header))
