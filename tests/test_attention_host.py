"""The paged-cache operators (include/native_hip_attention.h) as far as no GPU is needed: the entry points are there, their
refusals, which tiles and rows a launch reads, tables that name no block."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_every_declared_symbol(pkg, lib):
    header = open(os.path.join(ROOT, "include", "native_hip_attention.h")).read()
    declared = set(re.findall(r"\b(lnh_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", " ", header, flags=re.S)))
    assert declared == set(lib._paged_signatures)
    for name in declared:
        assert hasattr(lib, name), name


def test_structures_have_the_header_s_layout(pkg, tmp_path):
    import ctypes as C
    src, out = tmp_path / "layout.c", tmp_path / "layout"
    fields = [("lnh_kv_cache", pkg.KvCache), ("lnh_kv_seqs", pkg.KvSeqs)]
    lines = ["printf(\"%%zu\\n\", sizeof(%s));" % n for n, _ in fields]
    lines += ["printf(\"%%zu\\n\", offsetof(%s, %s));" % (n, f[0]) for n, s in fields for f in s._fields_]
    src.write_text('#include <stdio.h>\n#include "%s/include/native_hip_attention.h"\nint main(void) { %s return 0; }\n' % (ROOT, " ".join(lines)))
    cc = shutil.which(os.environ.get("CC", "gcc"))
    if cc is None:
        pytest.skip("no host C compiler")
    subprocess.run([cc, "-std=c99", "-Wall", "-Wextra", "-Werror", str(src), "-o", str(out)], check=True)
    want = [C.sizeof(s) for _, s in fields] + [getattr(s, f[0]).offset for _, s in fields for f in s._fields_]
    assert [int(x) for x in subprocess.run([str(out)], capture_output=True, text=True, check=True).stdout.split()] == want


def test_no_executor_is_an_error(lib):
    assert lib.lnh_kv_store_device(None, None, None, 0, None, 0, None, 0, None) == 1
    assert lib.lnh_attn_device(None, None, None, 0, 1, None, 0, None, 0, 1.0, 0, 0, 0, 1.0, None) == 1
    assert lib.lnh_kv_evict_device(None, None, None, 0, 1, 0, 0, 0, None, 0, None, None) == 1


def test_host_parts(tmp_path):
    """tests/cpp/attn_parts.cpp, built by the host compiler alone."""
    cxx = shutil.which(os.environ.get("CXX", "g++"))
    if cxx is None:
        pytest.skip("no host C++ compiler")
    out = tmp_path / "attn_parts"
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", os.path.join(ROOT, "tests", "cpp", "attn_parts.cpp"), "-o", str(out)],
                   check=True)
    r = subprocess.run([str(out)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout + r.stderr
