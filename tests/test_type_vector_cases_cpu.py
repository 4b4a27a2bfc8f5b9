"""Fixed cases of the type vectors' kernels on the emulated device (tests/emu/type_vector_cases.py)."""
import os
import subprocess
import sys

import pytest

RUNNER = os.path.join(os.path.dirname(os.path.abspath(__file__)), "emu", "type_vector_cases.py")


@pytest.mark.parametrize("name", ["numbers_beside_a_state", "many_tiles"])
def test_case(name):
    p = subprocess.run([sys.executable, RUNNER, name], stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                       text=True, timeout=600)
    assert p.returncode == 0 and name + " passed" in p.stdout, p.stdout[-3000:]


@pytest.mark.parametrize("name,passed", [("views", 2), ("rounds", 19)])
def test_device_tests_on_the_emulated_device(name, passed):
    """What the device tests ask of the functions; times and what needs autograd are left to the device."""
    here = os.path.dirname(RUNNER)
    p = subprocess.run([sys.executable, os.path.join(here, "gpu_tests_on_fake_device.py"),
                        os.path.join(os.path.dirname(here), "test_type_vector_%s_gpu.py" % name), "-m", "gpu", "-q",
                        "-k", "not time"],
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=1200)
    assert p.returncode == 0 and "%d passed" % passed in p.stdout, p.stdout[-3000:]


def test_the_contracting_build_fuses_products_and_sums():
    """EMU_CONTRACT=1 is for checks under fused multiply-adds: its results are not those of the build without."""
    lines = []
    for env in ({}, {"EMU_CONTRACT": "1"}):
        p = subprocess.run([sys.executable, RUNNER, "digest"], env=dict(os.environ, **env), stdout=subprocess.PIPE,
                           stderr=subprocess.STDOUT, text=True, timeout=1500)
        assert p.returncode == 0, p.stdout[-3000:]
        lines.append(p.stdout.splitlines())
    for plain, contracted in zip(lines[0][:2], lines[1][:2]):
        assert plain.split()[0] == contracted.split()[0] and plain != contracted
