"""Overlapping arrays are refused by the beam-search entry points before anything is launched."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "gemma4.pas_b200")


def test_overlaps(tmp_path, g4):
    exe = str(tmp_path / "beam_overlaps")
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run(["g++", "-std=c++17", "-x", "c++", "-O0", "-I", os.path.join(ROOT, "include"), "-I", f"{cuda}/include",
                    os.path.join(ROOT, "tests", "cpp", "beam_overlaps.cpp"), "-o", exe, "-L", PKG, "-lg4sampler",
                    f"-Wl,-rpath,{PKG}", "-L", f"{cuda}/lib64", "-lcudart", f"-Wl,-rpath,{cuda}/lib64", "-ldl", "-lpthread"],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
