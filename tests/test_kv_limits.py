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


def test_operators_refuse_gradients():
    """There is no backward pass: outside of no_grad() what requires a gradient is refused, not silently detached."""
    import pytest
    import torch

    from pegaflow_b200 import KVCache, chunk_attention, kv_read, kv_write

    def kv(grad=False):
        return torch.zeros((2, 4, 16, 2, 64), dtype=torch.bfloat16, requires_grad=grad)

    cache, x = KVCache.from_tensor(kv()), torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    y = x.clone().requires_grad_()
    slots, table = torch.zeros(3, dtype=torch.int64), torch.zeros((1, 4), dtype=torch.int32)
    q_start, kv_len = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    calls = [lambda: chunk_attention(y, cache, table, q_start, kv_len), lambda: kv_write(cache, y, x, slots),
             lambda: kv_write(cache, x, y, slots), lambda: kv_read(cache, table, q_start, out=(x, y)),
             lambda: chunk_attention(x, cache, table, q_start, kv_len, out=y)]
    for i, call in enumerate(calls):
        # Results are looked at behind the device, which a cache of the CPU does not have.
        words = "requires a gradient" if i < 3 else "requires a gradient|CUDA device"
        with pytest.raises(ValueError, match=words):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):
            call()
        with torch.inference_mode(), pytest.raises(ValueError, match="CUDA device"):
            call()
    with pytest.raises(ValueError, match="cannot require a gradient"):
        KVCache.from_tensor(kv(True))
    with torch.no_grad():
        KVCache.from_tensor(kv(True))


NO_TORCH = "import sys; sys.path.insert(0, '.'); sys.modules['torch'] = None\n"  # an import of it fails, and no spec is found


def run_python(code, *args):
    import sys

    return subprocess.run([sys.executable, "-c", code, *args], cwd=ROOT, capture_output=True, text=True, timeout=600)


def test_build_without_torch(native, tmp_path):
    """The library is for C and Rust callers too: without torch it is built as before, and the binding is left out."""
    out = run_python(NO_TORCH + "from pathlib import Path; from pegaflow_b200 import build as b\n"
                     "b.TORCH_BINDING = Path(sys.argv[1]) / 'x.so'; b.TORCH_STAMP = Path(sys.argv[1]) / 'x.stamp'\n"
                     "print(b.build()); print(list(Path(sys.argv[1]).iterdir()))", str(tmp_path))
    assert out.returncode == 0, out.stderr
    assert out.stdout.split() == [str(native.LIB_PATH), "[]"]


def test_import_without_torch(native):
    out = run_python(NO_TORCH + "from pegaflow_b200 import *\nprint(Layout.__name__, PegaEngine.__name__, 'kv_write' in globals())\n"
                     "import pegaflow_b200\ntry:\n    pegaflow_b200.kv_write\nexcept ImportError as e:\n    print('ImportError')")
    assert out.returncode == 0, out.stderr
    assert out.stdout.split() == ["Layout", "PegaEngine", "False", "ImportError"]
    import pegaflow_b200

    assert {"kv_write", "kv_read", "chunk_attention", "KVCache"} <= set(pegaflow_b200.__all__)


def test_import_beside_a_stand_in_for_torch(native):
    """A module named torch that somebody put together (to run without it) has no spec, and looking for one raises."""
    out = run_python("import sys, types; sys.path.insert(0, '.'); sys.modules['torch'] = types.ModuleType('torch')\n"
                     "from pegaflow_b200 import *\nfrom pegaflow_b200 import build as b\nprint(Layout.__name__, b._torch_home())")
    assert out.returncode == 0, out.stderr
    assert out.stdout.split() == ["Layout", "None"]


def test_binding_follows_the_installed_torch(native, tmp_path, monkeypatch):
    """A binding that another torch (or Python) was there for is built again, without being asked to."""
    import importlib.metadata

    from pegaflow_b200 import build as b

    built = tmp_path / "built"
    monkeypatch.setattr(b, "TORCH_BINDING", tmp_path / "x.so")
    monkeypatch.setattr(b, "TORCH_STAMP", tmp_path / "x.stamp", raising=False)
    monkeypatch.setattr(b, "_torch_command", lambda src, target, *_: ["sh", "-c", f"echo x >> {built}; touch {target}"])
    b.build()
    b.build()
    assert built.read_text() == "x\n"
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "9.9.9")
    b.build()
    b.build()
    assert built.read_text() == "x\nx\n"
