"""Overlapping arrays are refused by the beam-search entry points before anything is launched."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "gemma4.pas_b200")


@pytest.mark.parametrize("name", ["beam_overlaps", "beam_reorder_overlaps", "beam_pages_overlaps"])
def test_overlaps(tmp_path, g4, name):
    exe = str(tmp_path / name)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run(["g++", "-std=c++17", "-x", "c++", "-O1", "-I", os.path.join(ROOT, "include"), "-I", f"{cuda}/include",
                    os.path.join(ROOT, "tests", "cpp", f"{name}.cpp"), "-o", exe, "-L", PKG, "-lg4sampler",
                    f"-Wl,-rpath,{PKG}", "-L", f"{cuda}/lib64", "-lcudart", f"-Wl,-rpath,{cuda}/lib64", "-ldl", "-lpthread"],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
