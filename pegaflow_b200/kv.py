"""Paged-cache operators: what fills the cache that the transfers move, and what
reads it (pf_kv_* in include/pegaflow.h).

  KVCache            one layer's paged cache, 16-bit or 8-bit with fp32 scales
  kv_write           new tokens' K and V into cache slots, quantised on the way
  kv_read            the tokens of listed sequences back as dense K and V
  chunk_attention    attention of a chunk of new tokens over the cache (one
                     token each when decoding)

Each queues sm_100a kernels on a stream and returns: by default torch's current
stream of the cache's device, or ``stream`` (a cudaStream_t as int). Nothing is
synchronised or kept between calls, so they can be captured into CUDA graphs.
Sizes, types and strides are checked before anything is queued (ValueError, or
PegaError from the library); what only the device knows (slots, block ids,
lengths) is skipped where it is out of range, and reported through ``status``,
an int32 tensor that gets the bits BAD_BLOCK, BAD_LENGTH and TIMED_OUT (a wait
within a kernel ran out: the outputs are not valid) ORed into it.

A cache that a transfer loads, or that ``kv_write`` fills, is read by the others
as soon as their stream is behind it; the same tensors are registered with
``Layout.from_tensor`` (the scales as a layer of their own).
"""

from __future__ import annotations

import math
import struct
from ctypes import byref, c_uint64
from typing import Optional

import torch

from . import _native as N

BAD_BLOCK = N.PF_KV_BAD_BLOCK
BAD_LENGTH = N.PF_KV_BAD_LENGTH
TIMED_OUT = N.PF_KV_TIMED_OUT

_ROWS = {torch.bfloat16: N.PF_DTYPE_BF16, torch.float16: N.PF_DTYPE_FP16, torch.float32: N.PF_DTYPE_FP32}
_CACHE = {torch.bfloat16: N.PF_DTYPE_BF16, torch.float16: N.PF_DTYPE_FP16, torch.float8_e4m3fn: N.PF_DTYPE_E4M3,
          torch.uint8: N.PF_DTYPE_E4M3, torch.int8: N.PF_DTYPE_INT8}
_QUANTISED = (N.PF_DTYPE_E4M3, N.PF_DTYPE_INT8)
_pack_attention = struct.Struct("=QqqQqqQQqQQQQQQIIIIIIfIII").pack  # N.KvAttention, field by field
# The handle of torch's current stream of a device.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


class KVCache:
    """One layer's paged cache: addresses and strides of tensors that it keeps.

    ``key`` and ``value`` are views ``[num_blocks, block_size, heads, head_dim]``
    of any strides with a contiguous last axis: bf16 or fp16; or e4m3
    (``float8_e4m3fn``, or ``uint8`` holding its codes) or int8, with fp32
    scales that broadcast to ``[num_blocks, block_size, heads]``: one for each
    token and head, or shared (``[num_blocks, 1, 1]``: one for each block).
    """

    __slots__ = ("key", "value", "key_scale", "value_scale", "device", "dtype", "_c", "_ref", "_index",
                 "_heads", "_dim", "_quantised", "_scratch")

    def __init__(self, key: torch.Tensor, value: torch.Tensor, key_scale: Optional[torch.Tensor] = None,
                 value_scale: Optional[torch.Tensor] = None):
        _need(key.dim() == 4 and key.shape == value.shape, "key and value must both be [num_blocks, block_size, heads, "
              f"head_dim], not {tuple(key.shape)} and {tuple(value.shape)}")
        _need(key.dtype == value.dtype and key.dtype in _CACHE, "key and value must both be bfloat16, float16, "
              f"float8_e4m3fn, uint8 (e4m3 codes) or int8, not {key.dtype} and {value.dtype}")
        _need(key.shape[3] <= 1 or (key.stride(3) == 1 and value.stride(3) == 1),
              "the head_dim axis must be contiguous")
        code = _CACHE[key.dtype]
        scales = [key_scale, value_scale]
        if code in _QUANTISED:
            _need(key_scale is not None and value_scale is not None, f"a cache of {key.dtype} needs key and value scales")
            for i, s in enumerate(scales):
                _need(s.dtype == torch.float32, f"scales must be float32, not {s.dtype}")
                _need(s.dim() <= 3, "scales must broadcast to [num_blocks, block_size, heads]")
                try:
                    scales[i] = s.expand(key.shape[:3])
                except RuntimeError:
                    raise ValueError(f"scales of {tuple(s.shape)} do not broadcast to [num_blocks, block_size, heads] "
                                     f"= {tuple(key.shape[:3])}") from None
        else:
            _need(key_scale is None and value_scale is None, f"a cache of {key.dtype} has no scales")
        tensors = [t for t in (key, value, *scales) if t is not None]
        _need(all(t.device == key.device for t in tensors), "the cache's tensors must be on one device")
        self.key, self.value, self.key_scale, self.value_scale = key, value, *scales
        self.device, self.dtype = key.device, key.dtype
        # get_device(): -1 on the CPU, which every operator refuses.
        self._index = key.get_device()

        def side(t, s):
            b, o, h, _ = t.stride()
            return N.KvSide(t.data_ptr(), s.data_ptr() if s is not None else 0, b, o, h,
                            *(s.stride() if s is not None else (0, 0, 0)))

        self._c = N.KvCache(side(key, scales[0]), side(value, scales[1]), key.shape[0], key.shape[1], key.shape[2],
                            key.shape[3], code)
        self._ref = byref(self._c)
        self._heads, self._dim, self._quantised = key.shape[2], key.shape[3], code in _QUANTISED
        self._scratch = {}  # sizes of an attention call -> bytes of its workspace

    @staticmethod
    def from_tensor(t: torch.Tensor, scale: Optional[torch.Tensor] = None) -> "KVCache":
        """The cache in one tensor: KV-first ``[2, num_blocks, block_size, heads,
        head_dim]``, else blocks-first ``[num_blocks, 2, ...]``, with scales of
        the same leading axes (``[2, num_blocks, block_size, heads]``; axes of 1
        are shared), as ``Layout.from_tensor`` tells them apart. A scale of
        ``[num_blocks, 1]`` or ``[num_blocks]`` is one for each block, K and V."""
        _need(t.dim() == 5 and 2 in (t.shape[0], t.shape[1]),
              f"expected [2, num_blocks, ...] or [num_blocks, 2, block_size, heads, head_dim], not {tuple(t.shape)}")
        axis = 0 if t.shape[0] == 2 else 1
        if scale is not None and scale.dim() <= 2:
            s = scale.reshape(-1, 1, 1)
            ks = vs = s
        elif scale is not None:
            _need(scale.dim() == 4 and scale.shape[axis] == 2, "scales must have the tensor's leading axes")
            ks, vs = scale.select(axis, 0), scale.select(axis, 1)
        else:
            ks = vs = None
        return KVCache(t.select(axis, 0), t.select(axis, 1), ks, vs)

    @staticmethod
    def from_token_major(key: torch.Tensor, value: torch.Tensor, page_size: int,
                         key_scale: Optional[torch.Tensor] = None,
                         value_scale: Optional[torch.Tensor] = None) -> "KVCache":
        """Token-major K and V buffers ``[slots, heads, head_dim]`` whose pages of
        ``page_size`` tokens are the blocks (``Layout.from_token_major``), with
        scales ``[slots, heads]``."""
        _need(page_size > 0, "page_size must be > 0")
        _need(key.shape[0] % page_size == 0, f"KV slots ({key.shape[0]}) must be divisible by page_size ({page_size})")

        def paged(x):
            return None if x is None else x.unflatten(0, (-1, page_size))

        return KVCache(paged(key), paged(value), paged(key_scale), paged(value_scale))

    @property
    def num_blocks(self) -> int:
        return self._c.num_blocks

    @property
    def block_size(self) -> int:
        return self._c.block_size

    @property
    def heads(self) -> int:
        return self._c.heads

    @property
    def head_dim(self) -> int:
        return self._c.head_dim

    def _stream(self, stream: Optional[int]) -> int:
        if self._index < 0:
            raise ValueError("the cache must be on a CUDA device")
        return _raw_stream(self._index) if stream is None else stream

    def _new(self, shape: tuple, dtype: torch.dtype, stream: Optional[int]) -> torch.Tensor:
        """A new tensor that belongs to the stream that fills it."""
        if stream is None:
            return torch.empty(shape, dtype=dtype, device=self.device)
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, self.device)):
            return torch.empty(shape, dtype=dtype, device=self.device)

    def _ints(self, t: torch.Tensor, dtype: torch.dtype, dim: int, what: str) -> torch.Size:
        """The shape of a tensor of indices, lengths or offsets."""
        shape = t.shape
        if (t.dtype is not dtype or len(shape) != dim or t.get_device() != self._index
                or (shape[-1] > 1 and t.stride(-1) != 1)):
            raise ValueError(f"{what} must be {dtype} with {dim} axes, the last contiguous, on {self.device}")
        return shape

    def _status(self, status: Optional[torch.Tensor]) -> int:
        if status is None:
            return 0
        if status.dtype != torch.int32 or status.numel() != 1 or status.get_device() != self._index:
            raise ValueError(f"status must be one int32 on {self.device}")
        return status.data_ptr()

    def _rows(self, t: torch.Tensor, n: int, heads: int, what: str) -> tuple:
        """Address and strides of dense rows."""
        s = t.stride()
        if t.shape != (n, heads, self._dim) or t.get_device() != self._index or (s[2] != 1 and self._dim > 1):
            raise ValueError(f"{what} must be [{n}, {heads}, {self._dim}] with a contiguous last axis on "
                             f"{self.device}, not {tuple(t.shape)} with strides {s} on {t.device}")
        return t.data_ptr(), s[0], s[1]


def kv_write(cache: KVCache, key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor, *,
             given_scales: bool = False, status: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> None:
    """Writes ``key`` and ``value`` ``[n, heads, head_dim]`` (bf16, fp16 or fp32,
    any strides) into the cache at ``slots`` (int64 ``[n]``: block * block_size +
    offset; negative ones are skipped, the others distinct).

    A 16-bit cache takes the values rounded to its type. An 8-bit cache gets, for
    each token and head, scale = max|x| / 448 (e4m3) or / 127 (int8), at least
    2^-126, and codes = x / scale rounded to nearest; a row that holds a NaN or an
    infinity reads back as NaN. With ``given_scales`` the scales stay as they are
    (calibrated, or shared by a block), and values beyond them saturate."""
    n = key.shape[0]
    dtype = _ROWS.get(key.dtype)
    if dtype is None or value.dtype is not key.dtype:
        raise ValueError(f"key and value must both be bfloat16, float16 or float32, not {key.dtype} and {value.dtype}")
    heads = cache._heads
    k, kt, kh = cache._rows(key, n, heads, "key")
    v, vt, vh = cache._rows(value, n, heads, "value")
    if cache._ints(slots, torch.int64, 1, "slots")[0] != n:
        raise ValueError(f"{slots.shape[0]} slots for {n} tokens")
    rc = N.lib.pf_kv_write(cache._index, cache._ref, k, kt, kh, v, vt, vh, dtype, slots.data_ptr(), n,
                           1 if given_scales else 0, cache._status(status), cache._stream(stream))
    if rc:
        N.check(rc)


def kv_read(cache: KVCache, block_table: torch.Tensor, starts: torch.Tensor, total: Optional[int] = None, *,
            dtype: Optional[torch.dtype] = None, out: Optional[tuple] = None, status: Optional[torch.Tensor] = None,
            stream: Optional[int] = None) -> tuple:
    """Reads sequences' tokens back as dense ``(key, value)``, ``[total, heads,
    head_dim]`` each: token t of sequence s, on block ``block_table[s, t //
    block_size]`` (int32), becomes row ``starts[s] + t`` for every row of
    ``starts[s]`` to ``starts[s + 1]`` (int32, ``[n_seqs + 1]``, in order).

    ``total`` (at least ``starts[-1]``) and ``dtype`` (bf16, fp16, fp32; by
    default the cache's, bf16 for 8-bit codes) size new outputs; ``out`` gives
    them instead, and rows outside the sequences are left as they are. A token
    on a bad block reads as zeros."""
    seqs, blocks = cache._ints(block_table, torch.int32, 2, "block_table")
    if cache._ints(starts, torch.int32, 1, "starts")[0] != seqs + 1:
        raise ValueError(f"{starts.shape[0]} starts for {seqs} sequences: one more is needed")
    raw = cache._stream(stream)
    heads = cache._heads
    if out is None:
        if total is None or total < 0:
            raise ValueError("total, the rows of the result, must be given without out")
        if dtype is None:
            dtype = torch.bfloat16 if cache._quantised else cache.dtype
        code = _ROWS.get(dtype)
        if code is None:
            raise ValueError(f"dtype must be bfloat16, float16 or float32, not {dtype}")
        both = cache._new((2, total, heads, cache._dim), dtype, stream)
        key, value = both.unbind(0)
        n, t, h = total, heads * cache._dim, cache._dim
        k = (both.data_ptr(), t, h)
        v = (k[0] + n * t * both.element_size(), t, h)
    else:
        key, value = out
        n, code = key.shape[0], _ROWS.get(key.dtype)
        if code is None or value.dtype is not key.dtype:
            raise ValueError(f"outputs must both be bfloat16, float16 or float32, not {key.dtype} and {value.dtype}")
        if (total is not None and total != n) or (dtype is not None and dtype is not key.dtype):
            raise ValueError("total or dtype and out differ")
        k, v = cache._rows(key, n, heads, "key"), cache._rows(value, n, heads, "value")
    rc = N.lib.pf_kv_read(cache._index, cache._ref, block_table.data_ptr(), block_table.stride(0), blocks, seqs,
                          starts.data_ptr(), *k, *v, code, n, cache._status(status), raw)
    if rc:
        N.check(rc)
    return key, value


def chunk_attention(query: torch.Tensor, cache: KVCache, block_table: torch.Tensor, q_start: torch.Tensor,
                    kv_len: torch.Tensor, *, scale: Optional[float] = None, causal: bool = True, window: int = 0,
                    max_q: Optional[int] = None, max_kv: Optional[int] = None, out: Optional[torch.Tensor] = None,
                    return_lse: bool = False, status: Optional[torch.Tensor] = None, stream: Optional[int] = None):
    """Attention of each sequence's new tokens over its cached ones, themselves
    included (``kv_write`` them first).

    ``query`` ``[n_tokens, q_heads, head_dim]`` (bf16 or fp16) holds the chunks
    one after the other: sequence s has rows ``q_start[s]`` to ``q_start[s + 1]``
    (int32 ``[n_seqs + 1]``) and ``kv_len[s]`` (int32) tokens in the cache on the
    blocks ``block_table[s]`` (int32 ``[n_seqs, max_blocks]``), the chunk the last
    of them. A query at position p sees the tokens up to p (all of them without
    ``causal``), with ``window`` the last ``window`` of those only. ``q_heads`` is
    a multiple of the cache's heads; ``scale`` is 1 / sqrt(head_dim) by default.

    ``max_q`` and ``max_kv`` bound a sequence's new and cached tokens: they choose
    the kernel and how far it splits long sequences, never the result.

    Returns the output (``out``, or a new tensor like ``query``), and with
    ``return_lse`` the log of each row's sum of exponentials too, fp32
    ``[n_tokens, q_heads]``, with which outputs over parts of a sequence can be
    joined. A query that sees nothing gets zeros and -inf; rows outside the
    sequences are left as they are."""
    code = _ROWS.get(query.dtype)
    shape = query.shape
    if len(shape) != 3 or code is None:
        raise ValueError(f"query must be bfloat16 or float16 [n_tokens, q_heads, head_dim], not {query.dtype} "
                         f"{tuple(shape)}")
    n, heads, dim = shape
    q, qt, qh = cache._rows(query, n, heads, "query")
    seqs, blocks = cache._ints(block_table, torch.int32, 2, "block_table")
    if (cache._ints(q_start, torch.int32, 1, "q_start")[0] != seqs + 1
            or cache._ints(kv_len, torch.int32, 1, "kv_len")[0] != seqs):
        raise ValueError(f"{q_start.shape[0]} q_start and {kv_len.shape[0]} kv_len for {seqs} sequences")
    max_q, max_kv = max_q or 0, max_kv or 0
    if window < 0 or max_q < 0 or max_kv < 0:
        raise ValueError("window, max_q and max_kv cannot be negative")
    raw = cache._stream(stream)
    if out is None:
        out = cache._new(shape, query.dtype, stream)
        o, ot, oh = out.data_ptr(), heads * dim, dim
    else:
        if out.dtype is not query.dtype:
            raise ValueError(f"out must be {query.dtype}, not {out.dtype}")
        o, ot, oh = cache._rows(out, n, heads, "out")
    lse = cache._new((n, heads), torch.float32, stream) if return_lse else None
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    sizes = (n, seqs, blocks, heads, code, max_q, max_kv, window)
    need = cache._scratch.get(sizes)
    if need is None:
        need = _workspace(cache, sizes, scale)
    scratch = cache._new((need,), torch.uint8, stream) if need else None
    args = _pack_attention(q, qt, qh, o, ot, oh, lse.data_ptr() if return_lse else 0, block_table.data_ptr(),
                           block_table.stride(0), q_start.data_ptr(), kv_len.data_ptr(), cache._status(status),
                           scratch.data_ptr() if need else 0, need, n, seqs, blocks, heads, code, max_q, max_kv, scale,
                           1 if causal else 0, window, 0)
    rc = N.lib.pf_kv_attention_run(cache._index, cache._ref, args, raw)
    if rc:
        N.check(rc)
    return (out, lse) if return_lse else out


def _workspace(cache: KVCache, sizes: tuple, scale: float) -> int:
    n, seqs, blocks, heads, code, max_q, max_kv, window = sizes
    args = _pack_attention(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, n, seqs, blocks, heads, code, max_q, max_kv, scale, 1,
                           window, 0)
    need = c_uint64()
    N.check(N.lib.pf_kv_attention_workspace(cache._index, cache._ref, args, byref(need)))
    if len(cache._scratch) >= 1024:  # a server's sizes change with every step
        cache._scratch.clear()
    cache._scratch[sizes] = need.value
    return need.value
