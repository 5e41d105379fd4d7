"""The calls on sorted rows and adapters of the C++ face (sfnx/kernels.hpp) from a C++ host program, each against 64 bits on the host
(tests/cpp/sorted_rows.cpp)."""
import subprocess
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
PROG = Path(__file__).resolve().parent / "cpp" / "sorted_rows"


def test_cpp_sorted_rows():
    if not PROG.exists():
        from tests.cpp import build
        build.build()
    r = subprocess.run([str(PROG)], capture_output=True, text=True, timeout=100)
    print(r.stdout, r.stderr)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.strip().endswith("ok")
