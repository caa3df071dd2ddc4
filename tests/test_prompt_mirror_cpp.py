"""The operators on whole prompts through the C++ host-side mirror, by their own test program (built by __graft_entry__.build(), tests/cpp/Makefile)."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
BINARY = os.path.join(HERE, "cpp", "prompt_mirror_test")


def _run(mode: str):
    proc = subprocess.run([BINARY, mode], capture_output=True, text=True, timeout=120)
    assert proc.returncode == 0, proc.stdout + proc.stderr
    assert "all checks passed" in proc.stdout


def test_cpp_mirror_frequencies_and_refusals():
    if not os.path.exists(BINARY):
        subprocess.check_call(["make", "-C", os.path.join(HERE, "cpp"), "prompt_mirror_test"])
    _run("cpu")


@pytest.mark.gpu
def test_cpp_mirror_of_the_prompt_operators():
    if not os.path.exists(BINARY):
        pytest.fail("tests/cpp/prompt_mirror_test is not built (run __graft_entry__.build())")
    _run("gpu")
