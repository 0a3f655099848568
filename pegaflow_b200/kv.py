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
within a kernel ran out: the outputs are not valid) ORed into it. They are for
inference and have no backward pass: outside of ``torch.no_grad()`` tensors that
require a gradient are refused.

A cache that a transfer loads, or that ``kv_write`` fills, is read by the others
as soon as their stream is behind it; the same tensors are registered with
``Layout.from_tensor`` (the scales as a layer of their own).
"""

from __future__ import annotations

from ctypes import addressof
from typing import Optional

import torch

from . import _native as N  # loads the library that the binding is linked to

try:
    from . import _kv_torch as _ops
except ImportError as e:
    raise ImportError(f"{e}: build the torch binding with `python -m pegaflow_b200.build`") from e

BAD_BLOCK = N.PF_KV_BAD_BLOCK
BAD_LENGTH = N.PF_KV_BAD_LENGTH
TIMED_OUT = N.PF_KV_TIMED_OUT

_CACHE = {torch.bfloat16: N.PF_DTYPE_BF16, torch.float16: N.PF_DTYPE_FP16, torch.float8_e4m3fn: N.PF_DTYPE_E4M3,
          torch.uint8: N.PF_DTYPE_E4M3, torch.int8: N.PF_DTYPE_INT8}
_QUANTISED = (N.PF_DTYPE_E4M3, N.PF_DTYPE_INT8)


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

    __slots__ = ("key", "value", "key_scale", "value_scale", "device", "dtype", "_c", "_at", "_index")

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
        _need(not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)), "a cache cannot require a gradient, "
              "which these operators do not compute: make it under torch.no_grad(), or detach it")
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
        self._at = addressof(self._c)

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
    _ops.write(cache._at, cache._index, key, value, slots, given_scales, status, stream)


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
    return _ops.read(cache._at, cache._index, block_table, starts, total, dtype, out, status, stream)


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
    ``causal``), with ``window`` none at p - window or in front of it. ``q_heads`` is
    a multiple of the cache's heads; ``scale`` is 1 / sqrt(head_dim) by default.

    ``max_q`` and ``max_kv`` bound a sequence's new and cached tokens: they choose
    the kernel and how far it splits long sequences, and change the result by no
    more than rounding.

    Returns the output (``out``, or a new tensor like ``query``), and with
    ``return_lse`` the log of each row's sum of exponentials too, fp32
    ``[n_tokens, q_heads]``, with which outputs over parts of a sequence can be
    joined. A query that sees nothing gets zeros and -inf; rows outside the
    sequences are left as they are."""
    return _ops.attend(cache._at, cache._index, query, block_table, q_start, kv_len, scale, causal, window, max_q, max_kv,
                       out, return_lse, status, stream)
