"""Gradient clipping through the C++ host layers where gradients share a buffer, and from many threads: the programs build everywhere and
pass their checks on a GPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "ctensor_b200")
PROGRAMS = {"test_clip_slices": ("ctensor_host", ["host/include"]),
            "test_clip_slices_gen1": ("ctensor_gen1", ["host/gen1/include", "host/include"]),
            "test_clip_threads": ("ctensor_host", ["host/include"]),
            "test_clip_threads_gen1": ("ctensor_gen1", ["host/gen1/include", "host/include"])}


def _build(name):
    from ctensor_b200 import build as b
    b.build()
    b.build_host()
    b.build_gen1()
    library, includes = PROGRAMS[name]
    src = os.path.join(ROOT, "tests", "cpp", name + ".cpp")
    exe = os.path.join(ROOT, "tests", "cpp", name + ".bin")
    newest = max(os.path.getmtime(p) for p in (src, b.HOST_LIB, b.GEN1_LIB))
    if not os.path.exists(exe) or os.path.getmtime(exe) < newest:
        flags = [f for d in includes for f in ("-I", os.path.join(PKG, d))]
        subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-o", exe, src, *flags, "-L", PKG, "-l" + library, "-lctb200",
                               "-ldl", "-pthread", f"-Wl,-rpath,{PKG}"])
    return exe


@pytest.mark.parametrize("name", PROGRAMS)
def test_program_builds(name):
    assert os.path.exists(_build(name))


@pytest.mark.gpu
@pytest.mark.parametrize("name", PROGRAMS)
def test_program_passes(name):
    r = subprocess.run([_build(name)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "ALL PASSED" in r.stdout
