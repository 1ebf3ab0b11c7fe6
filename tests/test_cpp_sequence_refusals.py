"""What the C++ classes of the sequence operators refuse (tests/cpp/sequence_refusals.cpp)."""
import subprocess
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent


def test_refusals():
    out = HERE / "cpp" / "_build" / "sequence_refusals"
    out.parent.mkdir(parents=True, exist_ok=True)
    lib = ROOT / "lc_parallel_primitive_b200"
    subprocess.run(["g++", "-std=c++20", "-O2", f"-I{ROOT / 'include'}", "-I/usr/local/cuda/include",
                    str(HERE / "cpp" / "sequence_refusals.cpp"), "-o", str(out), f"-L{lib}", "-llcpp_b200",
                    f"-Wl,-rpath,{lib}", "-L/usr/local/cuda/lib64", "-lcudart", "-Wl,-rpath,/usr/local/cuda/lib64"],
                   check=True)
    r = subprocess.run([str(out)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
