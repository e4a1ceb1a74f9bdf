"""Paged key-value cache over the C ABI: keys and values quantised as they are written, read back, and attended to.

No counterpart in the reference, whose attention over compressed keys and values (TurboSparseAttentionReference,
runtime/backend/attention_ops.go:283-311; `turbo_sparse_attention` here) takes all of them from the host in every call.
All tensors are device memory, given by address; calls enqueue on a stream and return."""
from __future__ import annotations

import ctypes as C
import threading
from typing import Optional, Tuple, Union

from . import _lib
from ._lib import KvStrides, Stats
from .encoder import Runtime

FORMATS = {"f16": 0, "bf16": 1, "mx8": 2, "mx4": 3}
TYPES = {"f32": 0, "f16": 1, "bf16": 2}
PAGE_UNIT = 16


def _type(t: Union[str, int]) -> int:
    code = TYPES.get(t, t)
    if isinstance(code, str):
        raise ValueError(f"unsupported element type {t!r}; supported values are {', '.join(TYPES)}")
    return code


def _stream(stream: Optional[int]) -> Optional[int]:
    """None: the runtime's stream.  0, which is how CUDA and PyTorch name the default stream, is passed as its explicit
    handle, since a null handle means the runtime's stream to the library."""
    return 1 if stream == 0 else stream


def _strides(strides: Optional[Tuple[int, int, int, int]]):
    if strides is None:
        return None
    if len(strides) != 4:
        raise ValueError(f"strides are (key token, key head, value token, value head), got {strides!r}")
    return C.byref(KvStrides(*strides))


class _Results(threading.local):
    """Where a thread's calls leave launches and error: made once, which a call of a few microseconds notices."""

    def __init__(self):
        self.stats, self.err = Stats(), C.c_char_p()
        self.refs = C.byref(self.stats), C.byref(self.err)

    def done(self, rc: int) -> int:
        if rc:
            err, self.err = self.err, C.c_char_p()
            self.refs = C.byref(self.stats), C.byref(self.err)
            _lib.check(rc, err)
        return self.stats.kernel_launches


class KvCache:
    """`pages` pages of `page_size` tokens (a multiple of 16) x `kv_heads` heads of `head_dim` elements (32, 64, 96, 128,
    192 or 256), keys and values, on the runtime's device.  The caller hands pages out: row b of a page table
    [batch, max_pages] int32 lists the pages of sequence b in order.

    format: "f16" / "bf16" hold the rounded values, "mx8" e4m3 and "mx4" e2m1 codes with one power-of-two scale for every 32
    elements of a head's vector (the smallest that saturates nothing).

    Several threads may call one cache; what their calls enqueue is ordered by streams: attends of one cache one after the other,
    appends that overlap on different pages."""

    def __init__(self, rt: Runtime, pages: int, page_size: int, kv_heads: int, head_dim: int, format: str = "mx8"):
        if format not in FORMATS:
            raise ValueError(f"unsupported cache format {format!r}; supported values are {', '.join(FORMATS)}")
        self.rt = rt
        self.pages, self.page_size, self.kv_heads, self.head_dim, self.format = pages, page_size, kv_heads, head_dim, format
        self.handle = C.c_void_p()
        _lib.call("eos_b200_kv_cache_create", rt.handle, int(pages), int(page_size), int(kv_heads), int(head_dim),
                  FORMATS[format], C.byref(self.handle))
        rt._adopt(self)
        lib = _lib.lib()
        self._append, self._read = lib.eos_b200_kv_cache_append_device, lib.eos_b200_kv_cache_read_device
        self._attend = lib.eos_b200_kv_cache_attend_device
        self._results = _Results()

    @property
    def page_bytes(self) -> int:
        """Device bytes of one page (codes and scales of keys and values of all heads)."""
        return int(_lib.lib().eos_b200_kv_cache_page_bytes(self.handle))

    def append_device(self, d_key: int, d_value: int, type: Union[str, int], tokens: int, batch: int, d_page_table: int,
                      max_pages: int, d_starts: int, d_cu_tokens: Optional[int] = None,
                      strides: Optional[Tuple[int, int, int, int]] = None, stream: Optional[int] = None) -> int:
        """Writes new tokens: d_key, d_value [tokens, kv_heads, head_dim]; sequence b owns the rows d_cu_tokens[b] up to
        d_cu_tokens[b + 1] and writes them from position d_starts[b] on (None: one token per sequence).  strides: elements
        between (key tokens, key heads, value tokens, value heads).  Returns kernels launched."""
        r = self._results
        return r.done(self._append(self.handle, d_key, d_value, _type(type), tokens,
                                   _strides(strides), batch, d_page_table, max_pages, d_starts, d_cu_tokens, _stream(stream),
                                   *r.refs))

    def read_device(self, d_key: int, d_value: int, type: Union[str, int], tokens: int, batch: int, d_page_table: int,
                    max_pages: int, d_starts: int, d_cu_tokens: Optional[int] = None,
                    strides: Optional[Tuple[int, int, int, int]] = None, stream: Optional[int] = None) -> int:
        """The inverse of append_device with the same arguments: d_key, d_value receive the cached values.  Rows behind
        the last sequence are left as they were."""
        r = self._results
        return r.done(self._read(self.handle, d_key, d_value, _type(type), tokens,
                                 _strides(strides), batch, d_page_table, max_pages, d_starts, d_cu_tokens, _stream(stream),
                                 *r.refs))

    def attend_device(self, d_query: int, type: Union[str, int], q_heads: int, batch: int, d_page_table: int, max_pages: int,
                      d_lengths: int, d_out: int, scale: float, window: int = 0, d_lse: Optional[int] = None,
                      query_strides: Tuple[int, int] = (0, 0), stream: Optional[int] = None) -> int:
        """One new token per sequence: query [batch, q_heads, head_dim] attends to the last `window` (0: all) of
        d_lengths[b] cached positions; out [batch, q_heads, head_dim] of the query's type, d_lse [batch, q_heads] fp32 the
        logarithm of the softmax denominators.  Query head i reads key head i // (q_heads // kv_heads).  query_strides:
        elements between sequences and between heads, 0: contiguous.  Returns kernels launched."""
        if len(query_strides) != 2:
            raise ValueError(f"query_strides are (sequence, head), got {query_strides!r}")
        r = self._results
        return r.done(self._attend(self.handle, d_query, _type(type), q_heads, query_strides[0], query_strides[1], batch,
                                   d_page_table, max_pages, d_lengths, scale, window, d_out, d_lse, _stream(stream), *r.refs))

    def sync(self, stream: Optional[int] = None) -> None:
        """Waits for the stream; raises EosB200DeviceStatusError if a kernel met a page, position or length out of range."""
        _lib.call("eos_b200_kv_cache_sync", self.handle, _stream(stream))

    def close(self) -> None:
        if self.handle:
            _lib.lib().eos_b200_kv_cache_destroy(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
