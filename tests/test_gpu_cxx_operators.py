"""The C++ face of the drafted-token, page, norm and epilogue calls, run on the device against
formulas on the host (tests/cxx/operators_run.cpp)."""
import os
import shutil
import subprocess

import pytest

import reef_amd

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_operator_calls_on_the_device(tmp_path):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reef_amd.lib()  # the library must be built
    print("\n[case] C++ operators", flush=True)
    exe = tmp_path / "operators_run"
    libdir = os.path.dirname(reef_amd.LIB_PATH)
    cmd = ["g++", "-std=c++17", "-O1", "-ffp-contract=off", "-Wall", "-Wextra", "-Werror",
           "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"), "-isystem", "/opt/rocm/include",
           os.path.join(ROOT, "tests", "cxx", "operators_run.cpp"), "-L", libdir, "-lreef_hip",
           f"-Wl,-rpath,{libdir}", "-L/opt/rocm/lib", "-lamdhip64", "-Wl,-rpath,/opt/rocm/lib",
           "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    print(r.stdout, flush=True)
    assert r.returncode == 0, r.stdout + r.stderr
