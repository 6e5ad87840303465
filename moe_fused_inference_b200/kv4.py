"""Paged 4-bit KV cache: quantising write, read-back and attention over it.

``KV4Cache`` is one layer's pool of pages, each page holding ``page`` tokens of
every KV head; keys and values are MXFP4 (E2M1 values, one E8M0 code per 32
elements of a head), 4.25 bits an element — half of the FP8 cache of
``attn_decode`` — in the layout that include/moe_fp4.h describes.

* ``kv4_write`` quantises keys and values as they are written: the projections'
  rows as they are (bf16, fp16 or fp32, slices of a fused projection included).
* ``kv4_read`` gives tokens back as the values that the cache holds.
* ``kv4_attention`` is attention over the cache for any mix of sequences, from
  one token's decode step to whole prompts, with per-sequence lengths held on
  the device (nothing waits for the host: every call can be captured).

No reference counterpart: the reference holds one sequence's FP8 cache in one
buffer (runtime/model_runner_v2.py:39, src/ext/mxfp4_decode.cu:352-490).
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib

__all__ = ["KV4Cache", "kv4_write", "kv4_read", "kv4_attention", "attention_workspace"]

_DT = {torch.float32: _lib.MFI_F32, torch.float16: _lib.MFI_F16, torch.bfloat16: _lib.MFI_BF16}
_QT = (torch.bfloat16, torch.float16)
TILE = 16


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _stream(index: int) -> int:
    """The current stream of a device, without making a Stream object (these
    calls are a few microseconds of host time in all, 2 of them for that)."""
    return torch._C._cuda_getCurrentRawStream(index)


def _device() -> int:
    """The current device's index, without torch's own look at its initialisation.
    Launches, the error flag and the kernels' attributes belong to the current
    device: where the tensors are on another one, an entry point calls itself
    under ``torch.cuda.device``."""
    return torch._C._cuda_getDevice()


class KV4Cache:
    """A pool of pages.  ``data`` is uint8 (num_pages, kv_heads, page // 16,
    17 * head_dim); token slot ``s`` is token ``s % page`` of page ``s // page``."""

    def __init__(self, num_pages: int, page: int, kv_heads: int, head_dim: int, device="cuda"):
        _check(head_dim in (64, 128), "head_dim must be 64 or 128")
        _check(page > 0 and page % TILE == 0, "page must be a positive multiple of 16 tokens")
        _check(num_pages > 0 and kv_heads > 0, "num_pages and kv_heads must be positive")
        self._set(torch.zeros((num_pages, kv_heads, page // TILE, 17 * head_dim),
                              dtype=torch.uint8, device=device))

    @classmethod
    def wrap(cls, data: torch.Tensor) -> "KV4Cache":
        """The cache over existing memory (one layer of a larger allocation)."""
        _check(data.dim() == 4 and data.dtype == torch.uint8 and data.is_contiguous(),
               "data must be a contiguous uint8 tensor (num_pages, kv_heads, page // 16, 17 * head_dim)")
        _check(data.shape[3] in (17 * 64, 17 * 128), "head_dim must be 64 or 128")
        _check(data.numel() > 0, "the pool has no pages")
        _check(data.data_ptr() % 16 == 0, "data must be 16-byte aligned")
        self = cls.__new__(cls)
        self._set(data)
        return self

    def _set(self, data):
        self.data = data
        self.device = data.device
        self.vector = (data.shape[1], data.shape[3] // 17)   # of a token: heads, elements
        self.num_pages, self.kv_heads = data.shape[0], data.shape[1]
        self.page, self.head_dim = data.shape[2] * TILE, data.shape[3] // 17

    @property
    def capacity(self) -> int:
        """Tokens of the pool."""
        return self.num_pages * self.page


def _check_slots(slots, T, cache):
    _check(slots.is_cuda and slots.device == cache.device and slots.dtype == torch.int64
           and slots.dim() == 1, "slots must be a 1-D int64 tensor on the cache's device")
    _check(slots.shape[0] == T, "slots must have one entry per token")


def kv4_write(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise k, v (T, kv_heads, head_dim) into the tokens ``slots`` (int64
    (T,)) of the pool.  A negative slot skips its row (padding); a slot past
    the pool is skipped too and reported through the device error flag.  Slots
    of one call must differ.  k and v share a type (bf16, fp16 or fp32); rows
    and heads may have any stride, elements are contiguous.  A block with a
    value that is not finite reads back as NaN."""
    lib = _lib.load()
    dev, shape = cache.device, k.shape
    if not (k.is_cuda and k.device == dev and v.device == dev and slots.device == dev
            and k.dtype in _DT and v.dtype == k.dtype and len(shape) == 3 and v.shape == shape
            and shape[1:] == cache.vector and slots.dtype == torch.int64
            and slots.shape == shape[:1]):
        _check(k.is_cuda and v.is_cuda and cache.data.is_cuda, "tensors must be cuda")
        _check(k.device == dev and v.device == dev, "k and v must be on the cache's device")
        _check(k.dtype in _DT and v.dtype == k.dtype, "k and v must both be bfloat16, float16 or float32")
        _check(len(shape) == 3 and v.shape == shape and shape[1:] == cache.vector,
               "k and v must be (T, kv_heads, head_dim) of the cache")
        _check_slots(slots, shape[0], cache)
    if dev.index != _device():
        with torch.cuda.device(dev):
            return kv4_write(cache, k, v, slots)
    T = shape[0]
    if T == 0:
        return
    ks, vs = k.stride(), v.stride()
    if ks[2] != 1:
        k = k.contiguous()
        ks = k.stride()
    if vs[2] != 1:
        v = v.contiguous()
        vs = v.stride()
    if not slots.is_contiguous():
        slots = slots.contiguous()
    st = lib.mfi_kv4_write(
        k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], _DT[k.dtype],
        cache.data.data_ptr(), slots.data_ptr(), T, cache.kv_heads, cache.head_dim, cache.page,
        cache.num_pages, _stream(dev.index))
    _lib.check(st, "kv4_write")


def kv4_read(cache: KV4Cache, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """The tokens ``slots`` (int64 (T,)) of the pool as (k, v), each (T,
    kv_heads, head_dim) of ``dtype``, the held values rounded once to it.  A
    negative slot gives zeros; so does one past the pool, which is reported
    through the device error flag."""
    lib = _lib.load()
    dev = cache.device
    if not (slots.is_cuda and slots.device == dev and slots.dtype == torch.int64
            and slots.dim() == 1 and dtype in _DT):
        _check(cache.data.is_cuda, "tensors must be cuda")
        _check(dtype in _DT, "dtype must be bfloat16, float16 or float32")
        _check_slots(slots, slots.shape[0] if slots.dim() else 0, cache)
    if dev.index != _device():
        with torch.cuda.device(dev):
            return kv4_read(cache, slots, dtype)
    T = slots.shape[0]
    out = slots.new_empty((2, T, *cache.vector), dtype=dtype)
    if T:
        if not slots.is_contiguous():
            slots = slots.contiguous()
        k = out.data_ptr()
        st = lib.mfi_kv4_read(
            cache.data.data_ptr(), slots.data_ptr(), k, k + out.nbytes // 2, _DT[dtype], T,
            cache.kv_heads, cache.head_dim, cache.page, cache.num_pages, _stream(dev.index))
        _lib.check(st, "kv4_read")
    return out.unbind(0)


def attention_workspace(num_seqs: int, heads: int, cache: KV4Cache, max_q: int = 1) -> torch.Tensor:
    """A workspace for ``kv4_attention`` calls of up to ``num_seqs`` sequences
    of up to ``max_q`` rows each, initialised on the current stream.  Calls
    leave it ready for the next; calls that may run at the same time need one
    each."""
    _check(cache.data.is_cuda, "the cache must be cuda")
    lib = _lib.load()
    n = int(lib.mfi_kv4_attn_workspace_bytes(num_seqs, heads, cache.kv_heads, cache.head_dim, max_q))
    _check(n > 0, "num_seqs and max_q must be positive and heads a positive multiple of kv_heads")
    dev = cache.device
    if dev.index != _device():
        with torch.cuda.device(dev):
            return attention_workspace(num_seqs, heads, cache, max_q)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    _lib.check(lib.mfi_kv4_attn_init_workspace(ws.data_ptr(), n, _stream(ws.device.index)),
               "kv4_attn_init_workspace")
    return ws


def kv4_attention(q: torch.Tensor, cache: KV4Cache, page_table: torch.Tensor,
                  kv_lens: torch.Tensor, cu_q: Optional[torch.Tensor] = None,
                  max_q: Optional[int] = None, scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None,
                  workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the rows q (T, heads, head_dim), bf16 or fp16, over the cache.

    ``page_table`` int32 (n, pages) and ``kv_lens`` int32 (n,): sequence i is
    the first kv_lens[i] tokens of its pages.  Its rows are cu_q[i] ..
    cu_q[i + 1] - 1 (int32 (n + 1,)), at most ``max_q`` (T if not given); without
    cu_q every sequence has T / n rows.  They are the last of its tokens: row r
    of R sees tokens 0 .. kv_lens[i] - R + r, and one that sees none gives
    zeros.  Query head h reads KV head h / (heads / kv_heads); ``scale`` is 1 /
    sqrt(head_dim) if not given.  Returns (T, heads, head_dim) of q's type; rows
    that no sequence owns are not written.

    Softmax weights are rounded to fp16 (a relative 2^-12) before they meet the
    values; scores and sums are fp32.  That makes the error of an fp16 output up
    to a third larger than rounding alone (decode rows with few strong tokens
    2%), of a bf16 output under 1%; include/moe_fp4.h gives the ranges of keys,
    values and weights.

    Page ids, lengths and row ranges are read on the device; what lies outside
    the pool, the table or q is reported through the device error flag (and read
    as page 0, cut to the table, or left out).  ``workspace``: from
    ``attention_workspace``; made for this call if not given."""
    lib = _lib.load()
    dev, shape = cache.device, q.shape
    if not (q.is_cuda and q.device == dev and page_table.device == dev and kv_lens.device == dev
            and q.dtype in _QT and len(shape) == 3 and shape[2] == cache.head_dim
            and shape[1] > 0 and shape[1] % cache.kv_heads == 0 and page_table.dtype == torch.int32
            and page_table.dim() == 2 and kv_lens.dtype == torch.int32
            and kv_lens.shape == page_table.shape[:1]):
        _check(q.is_cuda and cache.data.is_cuda and page_table.is_cuda and kv_lens.is_cuda,
               "tensors must be cuda")
        _check(q.device == dev and page_table.device == dev and kv_lens.device == dev,
               "tensors must be on one device")
        _check(q.dtype in _QT, "q must be bfloat16 or float16")
        _check(len(shape) == 3 and shape[2] == cache.head_dim, "q must be (T, heads, head_dim) of the cache")
        _check(shape[1] > 0 and shape[1] % cache.kv_heads == 0,
               "heads must be a positive multiple of kv_heads")
        _check(page_table.dtype == torch.int32 and page_table.dim() == 2, "page_table must be int32 (n, pages)")
        _check(False, "kv_lens must be int32 (n,)")
    if dev.index != _device():
        with torch.cuda.device(dev):
            return kv4_attention(q, cache, page_table, kv_lens, cu_q, max_q, scale, out, workspace)
    T, heads, D = shape
    n, width = page_table.shape
    if cu_q is None:
        _check(T % n == 0 if n else T == 0, "without cu_q every sequence has the same count of rows")
        max_q = T // n if n else 0
    else:
        _check(cu_q.device == dev and cu_q.dtype == torch.int32 and cu_q.shape == (n + 1,),
               "cu_q must be int32 (n + 1,) on q's device")
        if not cu_q.is_contiguous():
            cu_q = cu_q.contiguous()
        max_q = T if max_q is None else min(int(max_q), T)
        _check(max_q >= 0, "max_q must not be negative")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _check(out.shape == shape and out.dtype == q.dtype and out.device == dev
               and out.is_contiguous(), "out must be a contiguous tensor of q's shape, type and device")
    if T == 0 or n == 0 or max_q == 0:
        return out
    qs = q.stride()
    if qs[2] != 1:
        q = q.contiguous()
        qs = q.stride()
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    if not kv_lens.is_contiguous():
        kv_lens = kv_lens.contiguous()
    if workspace is None:
        workspace = attention_workspace(n, heads, cache, max_q)
    else:
        _check(workspace.device == dev and workspace.dtype == torch.uint8
               and workspace.is_contiguous(), "workspace must be a uint8 tensor on q's device")
    if scale is None:
        scale = D ** -0.5
    st = lib.mfi_kv4_attn(
        q.data_ptr(), _DT[q.dtype], qs[0], qs[1], cache.data.data_ptr(), page_table.data_ptr(),
        page_table.stride(0), kv_lens.data_ptr(), 0 if cu_q is None else cu_q.data_ptr(),
        out.data_ptr(), T, max_q, n, heads, cache.kv_heads, D, cache.page, cache.num_pages, width,
        scale, workspace.data_ptr(), workspace.numel(), _stream(dev.index))
    _lib.check(st, "kv4_attn")
    return out
