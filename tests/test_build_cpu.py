"""The build stands on the product's own sources: nothing of it reads the tests' emulation, and the
sources that do not compute type vectors do not see the helpers that do."""
import os
import re
import shutil
import stat
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "libmolgrid_amd", "csrc")
TYPE_VECTOR_SOURCES = ("embed.hip", "layer_norm.hip", "dropout.hip")

HIPCC = """#!%s
# stands in for the compiler: hands out the library that is there and notes what it was asked for
import os, shutil, sys
out = sys.argv[sys.argv.index("-o") + 1]
shutil.copyfile(%r, out)
with open(%r, "a") as f:
    f.write(" ".join(sys.argv[1:]) + "\\n")
"""


def headers_of(source, seen):
    """Names of the files in csrc that `source` includes, and those that they include."""
    with open(os.path.join(CSRC, source)) as f:
        names = re.findall(r'^\s*#include "([^"]+)"', f.read(), re.M)
    for name in names:
        if name not in seen and os.path.exists(os.path.join(CSRC, name)):
            seen.add(name)
            headers_of(name, seen)
    return seen


@pytest.mark.parametrize("source", sorted(f for f in os.listdir(CSRC) if f.endswith(".hip")))
def test_only_the_type_vectors_see_their_helpers(source):
    headers = headers_of(source, set())
    helpers = headers & {"element_types.h", "row_team.h"}
    assert bool(helpers) == (source in TYPE_VECTOR_SOURCES), (source, helpers)


def test_build_reads_nothing_of_the_emulation(tmp_path):
    """build() in a tree without tests/emu: every source goes to the compiler for gfx950, the oracle
    and the C++ program are built, the package is imported."""
    library = os.path.join(ROOT, "libmolgrid_amd", "libmolgrid_hip.so")
    tree, calls, hipcc = tmp_path / "tree", tmp_path / "calls", tmp_path / "hipcc"
    skip = shutil.ignore_patterns("__pycache__", "build", "*.so", "*.o")
    for part in ("libmolgrid_amd", "include", "oracle", os.path.join("tests", "cpp")):
        shutil.copytree(os.path.join(ROOT, part), str(tree / part), ignore=skip)
    shutil.copyfile(os.path.join(ROOT, "__graft_entry__.py"), str(tree / "__graft_entry__.py"))
    hipcc.write_text(HIPCC % (sys.executable, library, str(calls)))
    hipcc.chmod(hipcc.stat().st_mode | stat.S_IEXEC)
    r = subprocess.run([sys.executable, "-c", "import __graft_entry__; __graft_entry__.build()"],
                       cwd=str(tree), env=dict(os.environ, HIPCC=str(hipcc)), stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
    assert "libmolgrid_amd imported" in r.stdout
    compiled = calls.read_text().splitlines()
    for source in (f for f in os.listdir(CSRC) if f.endswith(".hip")):
        mine = [c for c in compiled if source in c]
        assert len(mine) == 1 and "--offload-arch=gfx950" in mine[0], (source, mine)
    assert os.path.exists(str(tree / "oracle" / "liboracle.so"))
