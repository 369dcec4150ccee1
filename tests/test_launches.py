"""What launches ask of the runtime, recorded on the CPU by a program whose own HIP calls stand in for the runtime's."""
from __future__ import annotations

import subprocess

import pytest

from conftest import PKG_DIR, ROOT

LIBDIR = PKG_DIR / "rt4_amd" / "lib"


@pytest.fixture(scope="module")
def recorder(tmp_path_factory):
    exe = tmp_path_factory.mktemp("launches") / "recorder"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-D__HIP_PLATFORM_AMD__", f"-I{ROOT / 'include'}", "-I/opt/rocm/include", "-rdynamic",
                    str(ROOT / "tests" / "launch_recorder.cpp"), f"-L{LIBDIR}", "-lrt4k", f"-Wl,-rpath,{LIBDIR}", "-L/opt/rocm/lib",
                    "-Wl,-rpath,/opt/rocm/lib", "-Wl,--allow-shlib-undefined", "-o", str(exe)], check=True)
    return exe


@pytest.mark.parametrize("case", ["gate4_lds", "norm_without_y"])
def test_launches(rt4, recorder, case):
    r = subprocess.run([str(recorder), case], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    assert r.stdout.startswith("launches ")
