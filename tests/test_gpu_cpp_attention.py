"""The C++ layer's attention operators on the GPU: tests/cpp/test_attention.cpp exits nonzero on
any failed check."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "quasarml_b200", "cpp", "_build", "test_attention")


@pytest.mark.gpu
def test_attention_program():
    assert os.path.exists(BIN), "build the C++ layer first (make -C quasarml_b200/cpp)"
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=600)
    print(r.stdout)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "failed 0" in r.stdout
