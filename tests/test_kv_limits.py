"""Sizes next to the limits of the paged-cache operators, and the package where torch is missing. No GPU."""

import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_stream_parts():
    """The streaming kernel's parts, up to the longest block table (tests/kv_stream_test.cpp)."""
    build = ROOT / "tests" / "_build"
    build.mkdir(exist_ok=True)
    exe = build / "kv_stream_test"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover=all",
                    f"-I{ROOT / 'include'}", f"-I{ROOT / 'pegaflow_b200' / 'csrc'}", "-I/usr/local/cuda/include",
                    str(ROOT / "tests" / "kv_stream_test.cpp"), "-o", str(exe)], check=True, capture_output=True, text=True)
    out = subprocess.run([str(exe), "4000"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout + out.stderr
