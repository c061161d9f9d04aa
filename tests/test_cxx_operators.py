"""The C++ face of the drafted-token, page, norm and epilogue calls compiles against the C
ABI and throws the engine's exceptions. Host-only: every call fails validation."""
import os
import shutil
import subprocess

import pytest

import reef_amd

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_operator_wrappers_throw(tmp_path):
    reef_amd.lib()  # the library must be built
    exe = tmp_path / "operators_check"
    libdir = os.path.dirname(reef_amd.LIB_PATH)
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__",
           "-I", os.path.join(ROOT, "include"), "-isystem", "/opt/rocm/include",
           os.path.join(ROOT, "tests", "cxx", "operators_check.cpp"),
           "-L", libdir, "-lreef_hip", f"-Wl,-rpath,{libdir}", "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    print(r.stdout)
    assert r.returncode == 0, r.stdout + r.stderr
