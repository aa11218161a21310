"""Which kernels a call of attention over the paged cache takes, and which calls no launch holds, as far as no GPU is needed."""
import os
import shutil
import subprocess

import pytest

from attn_path_cases import F16, F32, LISTS_MANY, LISTS_SHARED, LISTS_WHOLE, PARTS, Q4_0, SHARED

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    """tests/cpp/attn_paths.cpp, built by the host compiler alone."""
    cxx = shutil.which(os.environ.get("CXX", "g++"))
    if cxx is None:
        pytest.skip("no host C++ compiler")
    out = tmp_path_factory.mktemp("paths") / "attn_paths"
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", os.path.join(ROOT, "tests", "cpp", "attn_paths.cpp"), "-o", str(out)],
                   check=True)
    return str(out)


def test_host_parts(program):
    r = subprocess.run([program], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout + r.stderr


def paths(program, calls):
    """The paths of calls given as dicts: type, heads, heads_kv, dim, block, seqs, and what differs from one new token a sequence behind everything."""
    lines = []
    for c in calls:
        new = c.get("new", 1)
        lines.append(" ".join(str(x) for x in (c["type"], c["heads"], c["heads_kv"], c["dim"], c["block"], c["seqs"], c.get("tokens", c["seqs"] * new), new, c["len"],
                                                c.get("window", 0), c.get("sinks", 0), int(c.get("weights", False)), c.get("select", 0))))
    r = subprocess.run([program, "-"], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=60, check=True)
    out = r.stdout.strip().split("\n")
    assert len(out) == len(calls)
    return out


@pytest.mark.parametrize("type,heads,heads_kv,dim,seqs,length,path", [
    (F16, 32, 8, 128, 16, 700, "shares"), (F32, 32, 8, 128, 16, 200, "shares"), (F16, 14, 2, 64, 64, 1000, "shares"), (F16, 8, 1, 128, 128, 700, "shares"),
    (F16, 32, 8, 128, 16, 400, "whole"), (F32, 32, 8, 128, 16, 100, "whole"), (F16, 32, 8, 128, 1, 400, "whole"), (F16, 32, 8, 128, 32, 1000, "whole"),
    (F32, 32, 8, 128, 256, 700, "shares"), (F16, 32, 8, 128, 256, 700, "whole"), (Q4_0, 32, 8, 128, 16, 1000, "whole")])
def test_a_long_sequence_does_not_wait_for_one_workgroup(program, type, heads, heads_kv, dim, seqs, length, path):
    """Where a batch leaves half of the compute units idle, its longest sequence may be alone: it is shared out unless a workgroup has it done as soon."""
    assert paths(program, [dict(type=type, heads=heads, heads_kv=heads_kv, dim=dim, block=16, seqs=seqs, len=length)])[0].split()[0] == path


@pytest.mark.parametrize("name,calls,kernel", [("shares", SHARED, "shares"), ("parts", PARTS, "shares"), ("lists, whole", LISTS_WHOLE, "whole"),
                                               ("lists, shares", LISTS_SHARED, "shares"), ("lists, many rows", LISTS_MANY, "many")])
def test_calls_take_the_kernels_they_are_tested_for(program, name, calls, kernel):
    changes = [{}] if name != "shares" else [{}, dict(window=2500, sinks=40), dict(weights=True)]
    for change in changes:
        for call, path in zip(calls, paths(program, [dict(c, **change) for c in calls])):
            assert path.split()[0] == kernel, (call, change, path)
            if name == "parts":
                assert int(path.split("parts=")[1]) > 1, (call, path)
