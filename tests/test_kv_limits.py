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


def test_library_refuses_rows_that_a_tile_carries_past_an_int32(native):
    """Query rows are counted in int32, rounded up to tiles of 256: 2^31 - 2 of them on one KV head became a negative
    number of tiles, and nothing was computed. No address is followed and nothing is queued by this call."""
    from ctypes import byref, c_uint64

    N = native
    side = N.KvSide(4096, 0, 1024, 64, 64, 0, 0, 0)
    c = N.KvCache(side, side, 4, 16, 1, 64, N.PF_DTYPE_BF16)
    r, need = N.KvRows(4096, 128, 64), c_uint64()

    def answer(n_tokens):
        a = N.KvAttention(r, r, 0, 4096, 4, 4096, 4096, 0, 0, 0, n_tokens, 1, 4, 2, N.PF_DTYPE_BF16, 0, 0, 1.0, 1, 0)
        rc = N.lib.pf_kv_attention_workspace(0, byref(c), byref(a), byref(need))
        return rc == N.PF_ERR_INVALID_ARGUMENT and "too many query tokens" in N.lib.pf_last_error().decode()

    assert answer(2 ** 30 - 1) and answer(2 ** 30 - 2 ** 15 + 1)
    assert not answer(2 ** 30 - 2 ** 15)
