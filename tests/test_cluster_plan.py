"""How many clusters the device runs at once: a failed question is not an
answer.  CPU only: the question is the test's own."""
import os
import subprocess

from conftest import ROOT


def test_only_answers_are_kept(tmp_path):
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    exe = str(tmp_path / "ask_once")
    r = subprocess.run(["g++", "-std=c++17", "-I", os.path.join(cuda, "include"), "-I", os.path.join(ROOT, "voxtral.c_b200", "csrc"),
                        os.path.join(ROOT, "tests", "host", "ask_once.cpp"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
