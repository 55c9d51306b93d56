"""CPU: the arithmetic of va_attend_paged's shares (voltattn_amd/csrc/va_shares.hpp), which
tests/cpp/test_shares.cpp drives directly, the same code as the kernels': every unit of a batch in one
share, shares by age in their proportion, every tile of every block in one piece, in order, and of a block
that is cut one piece that begins and one that ends it."""
import subprocess
import tempfile
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_shares():
    with tempfile.TemporaryDirectory() as d:
        exe = Path(d) / "test_shares"
        subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                        "-I", str(ROOT / "voltattn_amd" / "csrc"), str(ROOT / "tests" / "cpp" / "test_shares.cpp"), "-o", str(exe)], check=True)
        r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr
        assert "shares: ok" in r.stdout
