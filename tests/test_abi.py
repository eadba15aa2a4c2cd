"""The C ABI library loads and exports every symbol include/prism_hip.h declares (no GPU calls)."""

import ctypes
import os
import subprocess

import pytest

import prism_hip


def test_library_exports_every_declared_symbol():
    assert os.path.exists(prism_hip.LIB_PATH), "build libprism_hip.so first (prism-inference_amd/build.py)"
    lib = ctypes.CDLL(prism_hip.LIB_PATH)
    declared = prism_hip.header_symbols()
    assert len(declared) >= 25
    missing = [s for s in declared if not hasattr(lib, s)]
    assert not missing, missing
    # The binding covers the whole declared surface.
    prism_hip.lib()
    bound = {name for name in declared if getattr(prism_hip.lib(), name).argtypes is not None}
    assert bound == set(declared)


def test_struct_layouts_match_the_reference_blocks():
    # tools/ternary/src/lib.rs:27-39 (292-byte Q8_K) and src/kernels.rs:528-535 (prepared Q8_0)
    assert prism_hip.Q8K_DTYPE.itemsize == 292
    assert prism_hip.Q8K_DTYPE.fields["values"][1] == 4
    assert prism_hip.Q8_DTYPE.itemsize == 40


def test_library_does_not_link_the_oracle():
    with open(prism_hip.LIB_PATH, "rb") as f:
        blob = f.read()
    assert b"liboracle" not in blob and b"po_matvec" not in blob


@pytest.mark.parametrize("compiler,standard", [("gcc", "c99"), ("gcc", "gnu99"), ("gcc", "c11"), ("g++", "c++11"), ("g++", "c++17")])
def test_header_compiles_in_strict_standards(tmp_path, compiler, standard):
    """Strict C99 and C++ take the header; both names of a cache's scales are one pointer, where the binding has it."""
    source = tmp_path / ("user.c" if compiler == "gcc" else "user.cpp")
    offset = {n: getattr(prism_hip.KvCache, n).offset for n in ("k_scale", "v_scale", "format")}
    source.write_text("#include <prism_hip.h>\n#include <stddef.h>\n"
                      "typedef char as_bound[offsetof(prism_kv_cache, k_scale) == %(k_scale)d && offsetof(prism_kv_cache, k_exponent) == %(k_scale)d &&\n"
                      "    offsetof(prism_kv_cache, v_scale) == %(v_scale)d && offsetof(prism_kv_cache, v_exponent) == %(v_scale)d &&\n"
                      "    offsetof(prism_kv_cache, format) == %(format)d ? 1 : -1];\n" % offset +
                      "int main(void) { as_bound a; prism_kv_cache c; c.k_scale = 0; c.v_exponent = 0; a[0] = 0; return a[0] + (c.k_scale != 0) + (c.v_exponent != 0); }\n")
    p = subprocess.run([compiler, "-std=" + standard, "-Wall", "-Wextra", "-pedantic-errors", "-I", os.path.dirname(prism_hip.HEADER),
                        "-fsyntax-only", str(source)], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, p.stderr
