"""The sequence operators through the C++ headers (tests/cpp/sequence_test.cpp)."""
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent


def build() -> Path:
    out = HERE / "cpp" / "_build" / "sequence_test"
    out.parent.mkdir(parents=True, exist_ok=True)
    lib = ROOT / "lc_parallel_primitive_b200"
    subprocess.run(["g++", "-std=c++20", "-O2", f"-I{ROOT / 'include'}", "-I/usr/local/cuda/include",
                    str(HERE / "cpp" / "sequence_test.cpp"), "-o", str(out), f"-L{lib}", "-llcpp_b200",
                    f"-Wl,-rpath,{lib}", "-L/usr/local/cuda/lib64", "-lcudart", "-Wl,-rpath,/usr/local/cuda/lib64"],
                   check=True)
    return out


def test_headers_compile():
    assert build().exists()


@pytest.mark.gpu
def test_headers_run(cuda):
    r = subprocess.run([str(build())], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr[-2000:]
    assert "OK: 0 failure(s)" in r.stdout
