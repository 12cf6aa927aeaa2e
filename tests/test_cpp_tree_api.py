"""The tree step of the C++ mirror (tests/cpp/tree_api_test.cpp): its cases
report themselves skipped without a GPU, and pass on one."""

import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BINARY = os.path.join(ROOT, "tests", "cpp", "tree_api_test")


def run(env=None):
    if not os.path.exists(BINARY):
        pytest.skip("tests/cpp/tree_api_test is not built (make -C tests/cpp)")
    r = subprocess.run([BINARY], capture_output=True, text=True, timeout=110, env=env)
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr[-4000:]
    return r.stdout


def test_cpp_tree_step_skips_without_a_gpu():
    assert "0 ran, 1 skipped, 0 failed" in run(dict(os.environ, HIP_VISIBLE_DEVICES=""))


@pytest.mark.gpu
def test_cpp_tree_step_passes_on_gpu():
    assert "1 ran, 0 skipped, 0 failed" in run()
