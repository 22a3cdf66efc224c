"""Tests of the reference's host are skipped where its sources are absent or
the folder is empty, and run where they are there."""
import os
import subprocess
import sys

from conftest import ROOT


def run(folder):
    env = dict(os.environ, VOX_REFERENCE_DIR=str(folder))
    return subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", os.path.join("tests", "test_integration.py"),
                           "-k", "hooks"], cwd=ROOT, env=env, capture_output=True, text=True)


def test_an_empty_folder_is_no_reference(tmp_path):
    for folder in (tmp_path, tmp_path / "absent"):
        r = run(folder)
        assert r.returncode == 0 and "1 skipped" in r.stdout, r.stdout


def test_sources_are_not_skipped(tmp_path):
    (tmp_path / "voxtral.c").write_text("int main(void) { return 0; }\n")
    r = run(tmp_path)
    assert r.returncode == 1 and "1 failed" in r.stdout, r.stdout   # its anchors are not there
