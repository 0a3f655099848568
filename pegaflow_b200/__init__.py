"""B200-native KV-cache block transfer path with PegaFlow's engine API.

Public surface (mirrors the reference's ``pegaflow.pegaflow`` module):
  PegaEngine, PyLoadState        in-process engine + shm load flag
  Executor, Layout, SaveSpec ... transfer executor (C ABI pf_executor_*)
  KVCache, kv_write, kv_read,    operators on the paged cache that is moved
  chunk_attention                (C ABI pf_kv_*)

The native library is loaded on first use of any of these names, so
``pegaflow_b200.build`` can run before the library exists. A missing or
broken library raises ImportError at that first use; there is no fallback.
"""

import importlib
import importlib.util

_EXPORTS = {
    "PegaEngine": ".engine",
    "PyLoadState": ".engine",
    "EngineRpcClient": ".client",
    "CudaIPCWrapper": ".ipc",
    "PegaError": "._native",
    "LIB_PATH": "._native",
    "Executor": ".transfer",
    "Layout": ".transfer",
    "LoadSpec": ".transfer",
    "SaveSpec": ".transfer",
    "P2PSpec": ".transfer",
    "PinnedBuffer": ".transfer",
    "refcopy_save": ".transfer",
    "refcopy_load": ".transfer",
    "segment_offset": ".transfer",
    "validate": ".transfer",
    "KVCache": ".kv",
    "kv_write": ".kv",
    "kv_read": ".kv",
    "chunk_attention": ".kv",
}


def _torch_found() -> bool:
    try:
        return importlib.util.find_spec("torch") is not None
    except ValueError:  # a module of that name that was not imported from anywhere: a stand-in
        return False


# `import *` takes the operators where torch is installed; by name they fail without it, with the reason.
__all__ = sorted(n for n, m in _EXPORTS.items() if m != ".kv" or _torch_found())


def __getattr__(name):
    if name in _EXPORTS:
        value = getattr(importlib.import_module(_EXPORTS[name], __name__), name)
        globals()[name] = value
        return value
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
