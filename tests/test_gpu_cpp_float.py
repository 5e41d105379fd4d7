"""The 8- and 16-bit experts' calls of the C++ face (sfnx/kernels.hpp) from a C++ host program, each against 64 bits on the host
and with pointer tables (tests/cpp/float_experts.cpp)."""
import subprocess
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
PROG = Path(__file__).resolve().parent / "cpp" / "float_experts"


def test_cpp_float_experts():
    if not PROG.exists():
        from tests.cpp import build
        build.build()
    r = subprocess.run([str(PROG)], capture_output=True, text=True, timeout=100)
    print(r.stdout, r.stderr)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.strip().endswith("ok")
