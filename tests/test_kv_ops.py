"""The paged-cache operators without a GPU: what they refuse, before anything
could be queued, and that the ctypes structs match the header."""

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent


def cache(dtype=torch.bfloat16, blocks=4, page=16, heads=2, dim=64, scale=None):
    from pegaflow_b200 import KVCache

    t = torch.zeros((2, blocks, page, heads, dim), dtype=dtype)
    if scale is None and dtype in (torch.int8, torch.uint8, torch.float8_e4m3fn):
        scale = torch.ones((2, blocks, page, heads))
    return KVCache.from_tensor(t, scale)


def rows(n=3, heads=2, dim=64, dtype=torch.bfloat16):
    return torch.zeros((n, heads, dim), dtype=dtype)


def test_struct_layouts_match_the_header(tmp_path):
    from pegaflow_b200 import _native as N

    pairs = {"pf_kv_side": N.KvSide, "pf_kv_cache": N.KvCache, "pf_kv_rows": N.KvRows, "pf_kv_attention": N.KvAttention}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "pegaflow.h"', "int main(void) {"]
    for name, cls in pairs.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    for line in out.splitlines():
        name, field, value = line.split()
        cls = pairs[name]
        want = ctypes.sizeof(cls) if field == "size" else getattr(cls, field).offset
        assert int(value) == want, line


@pytest.mark.parametrize("make, words", [
    (lambda K: K(torch.zeros(4, 16, 2, 64), torch.zeros(4, 16, 2, 64)), "bfloat16"),
    (lambda K: K(torch.zeros(4, 16, 2, 64).half(), torch.zeros(4, 16, 2, 32).half()), "num_blocks"),
    (lambda K: K(torch.zeros(4, 16, 64).half(), torch.zeros(4, 16, 64).half()), "num_blocks"),
    (lambda K: K(torch.zeros(4, 16, 2, 64).half(), torch.zeros(4, 16, 2, 64).bfloat16()), "both"),
    (lambda K: K(*[torch.zeros(4, 16, 64, 2).half().transpose(2, 3)] * 2), "contiguous"),
    (lambda K: K(*[torch.zeros(4, 16, 2, 64).to(torch.int8)] * 2), "needs key and value scales"),
    (lambda K: K(*[torch.zeros(4, 16, 2, 64).half()] * 2, torch.ones(4, 16, 2), torch.ones(4, 16, 2)), "no scales"),
    (lambda K: K(*[torch.zeros(4, 16, 2, 64).to(torch.int8)] * 2, *[torch.ones(4, 16, 2).half()] * 2), "float32"),
    (lambda K: K(*[torch.zeros(4, 16, 2, 64).to(torch.int8)] * 2, *[torch.ones(4, 8, 2)] * 2), "broadcast"),
    (lambda K: K.from_tensor(torch.zeros(3, 4, 16, 2, 64).half()), "expected"),
    (lambda K: K.from_token_major(torch.zeros(33, 2, 64).half(), torch.zeros(33, 2, 64).half(), 16), "divisible"),
])
def test_cache_refusals(make, words):
    from pegaflow_b200 import KVCache

    with pytest.raises(ValueError, match=words):
        make(KVCache)


def test_cache_views():
    from pegaflow_b200 import KVCache

    t = torch.zeros((5, 2, 16, 3, 64), dtype=torch.uint8)
    c = KVCache.from_tensor(t, torch.ones(5, 1))  # blocks-first, one scale for each block
    assert (c.num_blocks, c.block_size, c.heads, c.head_dim) == (5, 16, 3, 64)
    assert c._c.value.data - c._c.key.data == 16 * 3 * 64 and c._c.key.block_stride == 2 * 16 * 3 * 64
    assert (c._c.key.scale_block_stride, c._c.key.scale_token_stride, c._c.key.scale_head_stride) == (1, 0, 0)
    # Two blocks KV-first: the leading 2 is K and V, as Layout.from_tensor reads it.
    c = KVCache.from_tensor(torch.zeros((2, 2, 16, 3, 64), dtype=torch.float16))
    assert c._c.value.data - c._c.key.data == 2 * (16 * 3 * 64) * 2  # blocks, a block, bytes
    k = torch.zeros((64, 3, 64), dtype=torch.int8)
    c = KVCache.from_token_major(k, k, 4, torch.ones(64, 3), torch.ones(64, 3))
    assert (c.num_blocks, c.block_size) == (16, 4) and c._c.key.scale_token_stride == 3


def test_operators_refuse_the_cpu():
    from pegaflow_b200 import chunk_attention, kv_read, kv_write

    c, table, i32 = cache(), torch.zeros((1, 4), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA device"):
        kv_write(c, rows(), rows(), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA device"):
        kv_read(c, table, i32, 4)
    with pytest.raises(ValueError, match="CUDA device"):
        chunk_attention(rows(), c, table, i32, i32[:1])


@pytest.mark.parametrize("change, words", [
    (dict(key=rows(dim=32)), "key must be"),
    (dict(value=rows(n=2)), "value must be"),
    (dict(key=rows(dtype=torch.float64)), "bfloat16, float16 or float32"),
    (dict(value=rows(dtype=torch.float16)), "both"),
    (dict(slots=torch.zeros(3, dtype=torch.int32)), "slots must be"),
    (dict(slots=torch.zeros(6, dtype=torch.int64)[::2]), "slots must be"),
    (dict(slots=torch.zeros(4, dtype=torch.int64)), "4 slots for 3 tokens"),
    (dict(status=torch.zeros(1)), "status"),
])
def test_write_refusals(change, words):
    from pegaflow_b200 import kv_write

    args = dict(key=rows(), value=rows(), slots=torch.zeros(3, dtype=torch.int64)) | change
    with pytest.raises(ValueError, match=words):
        kv_write(cache(), **args)


@pytest.mark.parametrize("change, words", [
    (dict(block_table=torch.zeros((1, 4), dtype=torch.int64)), "block_table"),
    (dict(block_table=torch.zeros(4, dtype=torch.int32)), "block_table"),
    (dict(q_start=torch.zeros(3, dtype=torch.int32)), "q_start"),
    (dict(kv_len=torch.zeros(1, dtype=torch.int64)), "kv_len"),
    (dict(query=rows(dtype=torch.float32)[0]), "query"),
    (dict(query=rows(dim=128)), "query must be"),
    (dict(window=-1), "negative"),
])
def test_attention_refusals(change, words):
    from pegaflow_b200 import chunk_attention

    args = dict(query=rows(), cache=cache(), block_table=torch.zeros((1, 4), dtype=torch.int32),
                q_start=torch.zeros(2, dtype=torch.int32), kv_len=torch.zeros(1, dtype=torch.int32)) | change
    with pytest.raises(ValueError, match=words):
        chunk_attention(**args)


# The library's own checks, with addresses that are never followed.

def c_cache(N, dtype, dim=64, address=4096, heads=2, stride=None, scale=8192, scale_strides=(32, 2, 1)):
    row = dim if stride is None else stride
    side = N.KvSide(address, scale if dtype >= N.PF_DTYPE_E4M3 else 0, 16 * heads * row, heads * row, row, *scale_strides)
    return N.KvCache(side, side, 4, 16, heads, dim, dtype)


def attention(N, c, **change):
    r = N.KvRows(4096, 4 * c.head_dim, c.head_dim)
    a = N.KvAttention(r, r, 0, 4096, 4, 4096, 4096, 0, 0, 0, 3, 1, 4, 4, N.PF_DTYPE_BF16, 0, 0, 1.0, 1, 0)
    for k, v in change.items():
        setattr(a, k, v)
    return a


def message(N):
    return N.lib.pf_last_error().decode()


@pytest.mark.parametrize("make, words", [
    (lambda N: c_cache(N, N.PF_DTYPE_FP32), "cache dtype"),
    (lambda N: c_cache(N, N.PF_DTYPE_BF16, dim=0), "head_dim"),
    (lambda N: c_cache(N, N.PF_DTYPE_BF16, dim=272), "head_dim"),
    (lambda N: c_cache(N, N.PF_DTYPE_BF16, address=0), "no address"),
    (lambda N: c_cache(N, N.PF_DTYPE_BF16, address=4097), "not aligned"),
    (lambda N: c_cache(N, N.PF_DTYPE_INT8, scale=0), "needs scales"),
    (lambda N: c_cache(N, N.PF_DTYPE_INT8, scale=2), "scale address"),
    (lambda N: c_cache(N, N.PF_DTYPE_INT8, scale_strides=(1, 0, 0)), "shared scales"),
    (lambda N: c_cache(N, N.PF_DTYPE_BF16, heads=0), "heads"),
])
def test_library_refuses_caches(native, make, words):
    from ctypes import byref

    N = native
    c, r = make(N), (4096, 128, 64)
    rc = N.lib.pf_kv_write(0, byref(c), *r, *r, N.PF_DTYPE_BF16, 4096, 3, 0, 0, 0)
    assert rc == N.PF_ERR_INVALID_ARGUMENT and words in message(N), message(N)


def test_library_refuses_given_scales_of_16_bits(native):
    from ctypes import byref

    N = native
    c, r = c_cache(N, N.PF_DTYPE_BF16), (4096, 128, 64)
    rc = N.lib.pf_kv_write(0, byref(c), *r, *r, N.PF_DTYPE_BF16, 4096, 3, 1, 0, 0)
    assert rc == N.PF_ERR_INVALID_ARGUMENT and "no scales" in message(N)
    rc = N.lib.pf_kv_write(0, byref(c), *r, *r, N.PF_DTYPE_E4M3, 4096, 3, 0, 0, 0)
    assert rc == N.PF_ERR_INVALID_ARGUMENT and "rows must be" in message(N)
    assert N.lib.pf_kv_write(0, None, *r, *r, 0, 4096, 3, 0, 0, 0) == N.PF_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("make, change, words", [
    (lambda N: c_cache(N, N.PF_DTYPE_BF16, dim=72), {}, "multiple of 16"),
    (lambda N: c_cache(N, N.PF_DTYPE_BF16, dim=144), {}, "multiple of 16"),
    (lambda N: c_cache(N, N.PF_DTYPE_FP16), {}, "query's type"),
    (lambda N: c_cache(N, N.PF_DTYPE_BF16), {"dtype": 2}, "query must be"),
    (lambda N: c_cache(N, N.PF_DTYPE_BF16), {"q_heads": 3}, "multiple of the cache's heads"),
    (lambda N: c_cache(N, N.PF_DTYPE_BF16, stride=68), {}, "aligned to 16 bytes"),
    (lambda N: c_cache(N, N.PF_DTYPE_BF16, address=4104), {}, "aligned to 16 bytes"),
    (lambda N: c_cache(N, N.PF_DTYPE_BF16), {"q_start": 0}, "no q_start"),
    (lambda N: c_cache(N, N.PF_DTYPE_BF16), {"max_blocks": 1 << 28}, "block table"),
    (lambda N: c_cache(N, N.PF_DTYPE_BF16), {"n_tokens": 1 << 29}, "too many query tokens"),
])
def test_library_refuses_attention(native, make, change, words):
    from ctypes import byref

    N = native
    c = make(N)
    a = attention(N, c, **change)
    rc = N.lib.pf_kv_attention_run(0, byref(c), byref(a), 0)
    assert rc == N.PF_ERR_INVALID_ARGUMENT and words in message(N), message(N)


@pytest.mark.parametrize("axis", ["block_stride", "token_stride", "head_stride", "scale_block_stride",
                                  "scale_token_stride", "scale_head_stride"])
def test_library_refuses_negative_strides(native, axis):
    from ctypes import byref

    N = native
    c = c_cache(N, N.PF_DTYPE_INT8)
    setattr(c.value, axis, -getattr(c.value, axis))
    r = (4096, 128, 64)
    assert N.lib.pf_kv_write(0, byref(c), *r, *r, N.PF_DTYPE_BF16, 4096, 3, 0, 0, 0) == N.PF_ERR_INVALID_ARGUMENT
    assert "negative stride" in message(N)
    c = c_cache(N, N.PF_DTYPE_BF16)
    a = attention(N, c)
    a.query.head_stride = -64
    assert N.lib.pf_kv_attention_run(0, byref(c), byref(a), 0) == N.PF_ERR_INVALID_ARGUMENT
    assert "query has a negative stride" in message(N)


def test_library_refuses_results_that_share_their_place(native):
    from ctypes import byref

    N = native
    c = c_cache(N, N.PF_DTYPE_BF16)
    r, flat = (4096, 128, 64), (4096, 128, 0)
    rc = N.lib.pf_kv_read(0, byref(c), 4096, 4, 4, 1, 4096, *r, *flat, N.PF_DTYPE_BF16, 5, 0, 0)
    assert rc == N.PF_ERR_INVALID_ARGUMENT and "value has rows that share" in message(N)
    a = attention(N, c)
    a.out.token_stride = 0
    assert N.lib.pf_kv_attention_run(0, byref(c), byref(a), 0) == N.PF_ERR_INVALID_ARGUMENT
    assert "out has rows that share" in message(N)
    c.key.block_stride = 0
    rc = N.lib.pf_kv_write(0, byref(c), *r, *r, N.PF_DTYPE_BF16, 4096, 3, 0, 0, 0)
    assert rc == N.PF_ERR_INVALID_ARGUMENT and "cannot be written" in message(N)


@pytest.mark.parametrize("change, words", [
    ({"scale": float("nan")}, "scale must be finite"),
    ({"scale": float("inf")}, "scale must be finite"),
    ({"max_blocks": (1 << 31) // 16 - 4095}, "block table names more tokens"),
])
def test_library_refuses_scales_and_lengths(native, change, words):
    """A length that a tile's end would carry past an int32 is refused; the longest below it is not, for its sake."""
    from ctypes import byref

    N = native
    c = c_cache(N, N.PF_DTYPE_BF16)
    a = attention(N, c, **change)
    assert N.lib.pf_kv_attention_run(0, byref(c), byref(a), 0) == N.PF_ERR_INVALID_ARGUMENT
    assert words in message(N), message(N)
    a = attention(N, c, max_blocks=(1 << 31) // 16 - 4096, n_tokens=0)
    assert N.lib.pf_kv_attention_run(0, byref(c), byref(a), 0) == N.PF_OK


def test_library_refuses_unaligned_queries(native):
    from ctypes import byref

    N = native
    c = c_cache(N, N.PF_DTYPE_BF16)
    a = attention(N, c)
    a.query.token_stride = 257
    assert N.lib.pf_kv_attention_run(0, byref(c), byref(a), 0) == N.PF_ERR_INVALID_ARGUMENT
    assert "query and out rows" in message(N)


def test_empty_calls_need_nothing(native):
    """No tokens, no rows, no sequences: nothing is queued, no address is needed."""
    from ctypes import byref

    N = native
    c, r = c_cache(N, N.PF_DTYPE_BF16), (0, 0, 0)
    assert N.lib.pf_kv_write(0, byref(c), *r, *r, 0, None, 0, 0, 0, 0) == N.PF_OK
    assert N.lib.pf_kv_read(0, byref(c), None, 0, 0, 0, None, *r, *r, 0, 5, 0, 0) == N.PF_OK
    a = attention(N, c, n_tokens=0)
    assert N.lib.pf_kv_attention_run(0, byref(c), byref(a), 0) == N.PF_OK


def test_tile_spans():
    """The tile kernel's work shared among CTAs, replayed on the host (tests/kv_tiles_test.cpp)."""
    build = ROOT / "tests" / "_build"
    build.mkdir(exist_ok=True)
    exe = build / "kv_tiles_test"
    subprocess.run(["g++", "-O1", "-std=c++17", f"-I{ROOT / 'include'}", f"-I{ROOT / 'pegaflow_b200' / 'csrc'}",
                    "-I/usr/local/cuda/include", str(ROOT / "tests" / "kv_tiles_test.cpp"), "-o", str(exe)], check=True,
                   capture_output=True, text=True)
    out = subprocess.run([str(exe), "3000"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout
