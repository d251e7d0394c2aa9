"""The paged attention launchers on several devices, on the CPU: tests/paged_devices_check.cpp is linked with the library's
own objects of the two launchers and a fake CUDA runtime, and run."""
import importlib.util
import shutil
import subprocess

import pytest

from gptoss_b200 import capi


def test_shared_memory_limits_are_set_on_every_device(tmp_path):
    spec = importlib.util.spec_from_file_location("gptoss_build", capi.PKG / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    if not shutil.which("g++"):
        pytest.skip("g++ not found")
    if not (build.BUILD / "paged_attention_tc.o").exists():
        build.build()
    exe, include = tmp_path / "check", "/usr/local/cuda/include"
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(build.CSRC), "-I", include, "-o", str(exe),
                        str(capi.PKG.parent / "tests" / "paged_devices_check.cpp"), str(build.BUILD / "paged_attention.o"),
                        str(build.BUILD / "paged_attention_tc.o")], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.strip().endswith("OK"), out.stdout + out.stderr
