"""The library's host code against a stand-in for the CUDA runtime (tests/fake_runtime.h), compiled and run here."""

import os
import subprocess

from conftest import ROOT

CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


def _run(name, tmp_path):
    exe = str(tmp_path / name)
    here = os.path.join(ROOT, "tests")
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", f"-I{CUDA}/include", os.path.join(here, f"{name}.cc"), "-o", exe], check=True)
    done = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stderr


def test_a_failure_is_reported_once(tmp_path):
    _run("host_errors", tmp_path)


def test_shared_memory_limits_hold_between_threads(tmp_path):
    _run("host_shared_limit", tmp_path)
