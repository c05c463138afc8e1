"""Device code is compiled without packed fp32 instructions (some of their forms have given wrong results), whichever way it
is built: every object follows the Makefile, so that an object of earlier flags is not linked again, and the scripts that build
one object for a comparison use the same flags."""
import glob
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "dilabhelmholtzoct_amd", "csrc")
FLAG = "-Xclang -target-feature -Xclang -packed-fp32-ops"


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
def test_objects_follow_the_makefile():
    out = subprocess.run(["make", "-n", "-W", "Makefile", "-C", CSRC], check=True, capture_output=True, text=True).stdout
    compiled = [line for line in out.splitlines() if " -c " in line]
    sources = glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.cpp"))
    assert len(compiled) == len(sources) + 1  # (gemm.hip twice)
    assert all(FLAG in line for line in compiled)


def test_comparison_builds_use_the_flags():
    lines = []
    for f in glob.glob(os.path.join(ROOT, "scripts", "**", "*"), recursive=True):
        if f.endswith((".sh", ".py", ".hip")):
            with open(f) as src:
                lines += [(f, line) for line in src if "hipcc" in line and "--offload-arch" in line and "-shared" not in line]
    assert len(lines) >= 2
    for f, line in lines:
        assert FLAG in line, (f, line)


@pytest.mark.parametrize("source", sorted(os.path.basename(f) for f in glob.glob(os.path.join(CSRC, "*.hip"))))
def test_comparison_builds_find_their_headers(source):
    """build_ab_lib.sh compiles a source in a folder of its own: the headers beside it have to come along."""
    with open(os.path.join(CSRC, source)) as f:
        headers = [line.split('"')[1] for line in f if line.startswith('#include "') and "/" not in line]
    with open(os.path.join(ROOT, "scripts", "build_ab_lib.sh")) as f:
        script = f.read()
    for h in headers:
        assert h in script, h


def test_build_compiles_where_a_library_is_there(monkeypatch):
    """build() is the check that the sources compile: what is built already must not stand in for it."""
    import __graft_entry__ as entry
    calls = []
    monkeypatch.setattr(entry.subprocess, "run", lambda cmd, **kw: calls.append(cmd))
    entry.build()
    csrc = [c for c in calls if c[0] == "make" and any(str(a).endswith("csrc") for a in c)]
    assert len(csrc) == 1 and "-B" in csrc[0]
