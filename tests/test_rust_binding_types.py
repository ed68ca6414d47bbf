"""Every type that the generated Rust binding names is one that Rust has, that the file imports, or that it declares."""
import os
import re

import pytest

from tests.conftest import ROOT
from tests.test_abi_cpu import _load_generator

PRIMITIVE = {"i8", "i16", "i32", "i64", "u8", "u16", "u32", "u64", "usize", "isize", "f32", "f64", "bool"}


def test_types_of_the_binding_are_known():
    text = open(os.path.join(ROOT, "rust", "tract-rocm", "src", "ffi.rs")).read()
    imported = set(re.search(r"use std::os::raw::\{(.*?)\};", text).group(1).replace(" ", "").split(","))
    declared = set(re.findall(r"pub struct (\w+)", text))
    block = re.search(r'extern "C" \{\n.*?\n\}', text, flags=re.S).group(0)
    used = set()
    for args, ret in re.findall(r"pub fn \w+\((.*?)\) -> ([^;]+);", block):
        used |= {t.split()[-1] for t in [ret] + [a.split(": ")[1] for a in args.split(", ") if a]}
    assert len(used) > 8
    assert used <= PRIMITIVE | imported | declared, used - (PRIMITIVE | imported | declared)


def test_the_generator_refuses_a_type_it_does_not_know():
    gen = _load_generator()
    assert gen.rust_type("const int32_t *") == "*const i32"
    assert gen.rust_type("trocm_kv_cache *const *") == "*const *mut trocm_kv_cache"
    with pytest.raises(AssertionError):
        gen.rust_type("const int8_t *")
