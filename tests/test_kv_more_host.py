"""The rotated append, the read back, the 4-bit cache and chosen blocks as far as no GPU is needed: their refusals, the structure's layout, the packing's own
properties."""
import os
import shutil
import subprocess

import numpy as np
import pytest

from paged4 import pack, scale_of, split_buffer, to_buffer, unpack

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_structures_have_the_header_s_layout(pkg, tmp_path):
    import ctypes as C
    cc = shutil.which(os.environ.get("CC", "gcc"))
    if cc is None:
        pytest.skip("no host C compiler")
    src, out = tmp_path / "layout.c", tmp_path / "layout"
    lines = ["printf(\"%zu\\n\", sizeof(lnh_rope));"] + ["printf(\"%%zu\\n\", offsetof(lnh_rope, %s));" % f[0] for f in pkg.Rope._fields_]
    src.write_text('#include <stdio.h>\n#include "%s/include/native_hip_attention.h"\nint main(void) { %s return 0; }\n' % (ROOT, " ".join(lines)))
    subprocess.run([cc, "-std=c99", "-Wall", "-Wextra", "-Werror", str(src), "-o", str(out)], check=True)
    want = [C.sizeof(pkg.Rope)] + [getattr(pkg.Rope, f[0]).offset for f in pkg.Rope._fields_]
    assert [int(x) for x in subprocess.run([str(out)], capture_output=True, text=True, check=True).stdout.split()] == want


def test_no_executor_is_an_error(lib):
    assert lib.lnh_rope_table_device(None, 64, 1e4, 1.0, None, 1, None, 32, None) == 1
    assert lib.lnh_kv_append_device(None, None, None, 0, None, 0, None, 0, None, 0, None, 0, None, 0, None) == 1
    assert lib.lnh_kv_load_device(None, None, None, 0, None, 0, None, 0, None) == 1
    assert lib.lnh_kv_bounds_device(None, None, None, 0, None, None) == 1
    assert lib.lnh_attn_select_device(None, None, None, 0, 1, None, 1, 0, 1, None, 0, None, 0, 1.0, None, None) == 1


def test_host_parts(tmp_path):
    """tests/cpp/kv_parts.cpp, built by the host compiler alone."""
    cxx = shutil.which(os.environ.get("CXX", "g++"))
    if cxx is None:
        pytest.skip("no host C++ compiler")
    out = tmp_path / "kv_parts"
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", os.path.join(ROOT, "tests", "cpp", "kv_parts.cpp"), "-o", str(out)],
                   check=True)
    r = subprocess.run([str(out)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout + r.stderr


def test_packing(pkg):
    """What the tests pack: values are f16 exactly (unpack asserts it), within half a step unless they lie beyond seven of them, the same
    when packed again; the buffer is the header's."""
    rng = np.random.default_rng(0)
    for size in (1e-6, 1.0, 1e4):
        x = (rng.normal(0, size, (3, 2, 2, 5, 96))).astype(np.float32)
        words, scales = pack(x)
        y = unpack(words, scales).astype(np.float64)
        d = np.repeat(np.abs(scales.astype(np.float64)), 32, -1)
        sign = np.repeat(np.sign(scales.astype(np.float64)), 32, -1)
        inside = (x * sign < 7.5 * d) & (x * sign > -8.5 * d)
        assert np.all(np.abs(y - x)[inside] <= d[inside] / 2)
        assert inside.mean() > 0.97
        w2, s2 = pack(y.astype(np.float32))
        if size >= 1:  # an f16 below 2^-14 has fewer bits for the scale
            assert np.array_equal(w2, words) and np.array_equal(s2, scales)
        raw = to_buffer(x)
        assert raw.nbytes == pkg.q4_0_bytes(2, 2, 96, 5, 3)
        w3, s3 = split_buffer(raw, x.shape)
        assert np.array_equal(w3, words) and np.array_equal(s3, scales)


def test_a_word_by_hand():
    x = np.zeros(32, np.float32)
    x[0], x[1], x[2], x[7] = -8, 3, 7, -2.5  # d = 1: codes 0, 11, 15, 8 - 2 (a tie, to even)
    words, scales = pack(x)
    assert scales[0] == 1 and words[0] == 0 << 0 | 11 << 16 | 15 << 4 | 8 << 20 | 8 << 8 | 8 << 24 | 8 << 12 | 6 << 28
    assert list(words[1:]) == [0x88888888] * 3
    assert scale_of(np.full((1, 32), 1e9, np.float32))[0] == -8160
    assert np.isnan(scale_of(np.full((1, 32), np.inf, np.float32))[0])
