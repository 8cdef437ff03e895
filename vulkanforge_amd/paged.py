"""Host mirror of the paged cache: a pool of pages with reference counts, batches of sequences over it, and the calls that
fill and read it (``include/vfkv.h``, section "Paged cache").

Arguments are PyTorch device tensors; PyTorch only supplies memory and the stream.  Every compute method enqueues on
``stream`` (default: torch's current stream on the cache's device) and returns without synchronising.
"""
from __future__ import annotations

import ctypes as C
import math
from array import array
from dataclasses import dataclass
from typing import List, Optional, Sequence

import numpy as np

from . import _ffi
from .forward import Workspace
from .kv_cache import KvDtype

NO_PAGE = -1     # an entry of a page list or page table without a page
_TOP = 0xFFFFFFFF


def _fit(v: int) -> int:
    """``v``, or 2^32 - 1 where ctypes would wrap it to another number: no layer, page, size or count may be that one."""
    return v if 0 <= v <= _TOP else _TOP


@dataclass
class PagedKvConfig:
    n_layers: int
    n_kv_heads: int
    head_dim: int
    page_size: int
    n_pages: int
    dtype: KvDtype = KvDtype.F16


def _pages(values):
    """Page list (a sequence of whole numbers or a numpy array) -> unsigned 32-bit array; -1 becomes VFKV_NO_PAGE."""
    if isinstance(values, np.ndarray):
        if values.size and values.dtype.kind not in "iu":
            raise ValueError("pages are whole numbers")
        if values.size > 256:                            # (below, numpy's calls cost more than the list)
            if values.min() < -1 or values.max() > _ffi.NO_PAGE:
                raise ValueError("a page number does not fit")
            return np.ascontiguousarray(values.astype(np.uint32).reshape(-1))
        values = values.reshape(-1).tolist()
    try:
        return array("I", values)
    except TypeError:
        raise ValueError("pages are whole numbers") from None
    except OverflowError:
        pass
    try:
        return array("I", [_ffi.NO_PAGE if v == NO_PAGE else v for v in values])
    except OverflowError:
        raise ValueError("a page number does not fit") from None


def _addr(a) -> int:
    return a.buffer_info()[0] if isinstance(a, array) else a.__array_interface__["data"][0]


_IO: dict = {}           # torch dtype -> io_dtype, filled on first use (the package imports without torch)
_raw_stream = None


def _first_use() -> None:
    global _raw_stream
    import torch
    _IO.update({torch.float32: 0, torch.float16: 1})
    # the stream's handle without building a Stream object: a decode step calls this once per layer and operator
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    _raw_stream = raw or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _stream(stream, device=None) -> int:
    if stream is None:
        if _raw_stream is None:
            _first_use()
        if device is None:
            import torch
            device = torch.cuda.current_device()
        return _raw_stream(device)
    return stream if isinstance(stream, int) else stream.cuda_stream


class PagedKvCache:
    """K and V as [layer][page][kv_head][slot][d], and the reference counts of the pages.

    ``PagedKvCache(config)`` allocates on the current HIP device; ``k_buffer`` / ``v_buffer`` are device addresses of
    caller-owned memory instead (keep it alive); ``layout_only=True`` builds the page counting without buffers."""

    def __init__(self, config: PagedKvConfig, layout_only: bool = False, k_buffer: int = 0, v_buffer: int = 0):
        L = _ffi.lib()
        self.config = config
        self.kv_dtype = KvDtype(config.dtype)
        cfg = _ffi.PagesConfig(*(_fit(x) for x in (config.n_layers, config.n_kv_heads, config.head_dim, config.page_size,
                                                   config.n_pages)), int(self.kv_dtype))
        handle = C.c_void_p()
        if layout_only or k_buffer or v_buffer:
            _ffi.check(L.vfkv_pages_create_external(C.byref(cfg), k_buffer or None, v_buffer or None, C.byref(handle)))
        else:
            _ffi.check(L.vfkv_pages_create(C.byref(cfg), C.byref(handle)))
        self._h = handle
        self.device = None                               # index of the device the buffers are on
        if self.k_ptr:
            try:
                import torch
                if torch.cuda.is_available():
                    self.device = torch.cuda.current_device()
            except ImportError:
                pass

    def destroy(self) -> None:
        if getattr(self, "_h", None):
            _ffi.lib().vfkv_pages_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass

    @property
    def handle(self):
        return self._h

    # -- layout --
    @property
    def k_ptr(self) -> int:
        return int(_ffi.lib().vfkv_pages_k_ptr(self._h) or 0)

    @property
    def v_ptr(self) -> int:
        return int(_ffi.lib().vfkv_pages_v_ptr(self._h) or 0)

    def bytes_per_buffer(self) -> int:
        return int(_ffi.lib().vfkv_pages_bytes_per_buffer(self._h))

    def offset_bytes(self, layer: int, page: int) -> int:
        return int(_ffi.lib().vfkv_pages_offset_bytes(self._h, _fit(layer), _fit(page)))

    def pages_for(self, kv_len: int) -> int:
        """Pages a sequence of ``kv_len`` positions occupies."""
        return -(-kv_len // self.config.page_size)

    # -- page counting --
    @property
    def free_count(self) -> int:
        return int(_ffi.lib().vfkv_pages_free_count(self._h))

    def refcount(self, page: int) -> int:
        return int(_ffi.lib().vfkv_pages_refcount(self._h, _fit(page)))

    def alloc(self, n: int) -> List[int]:
        """The ``n`` lowest free pages; raises when fewer are free."""
        n = n if 0 <= n <= self.config.n_pages else _TOP                     # (more than there can be: the call says so)
        out = np.empty(n if 0 < n < _TOP else 1, np.uint32)
        _ffi.check(_ffi.lib().vfkv_pages_alloc(self._h, n, _addr(out)))
        return out[:n].tolist()

    def retain(self, pages: Sequence[int]) -> None:
        p = _pages(pages)
        _ffi.check(_ffi.lib().vfkv_pages_retain(self._h, _addr(p), len(p)))

    def release(self, pages: Sequence[int]) -> None:
        """One reference less per entry; pages without references are free (entries of -1 are skipped)."""
        p = _pages(pages)
        _ffi.check(_ffi.lib().vfkv_pages_release(self._h, _addr(p), len(p)))

    # -- pages on the device --
    def copy_pages(self, src: Sequence[int], dst: Sequence[int], rows: Optional[Sequence[int]] = None, stream=None) -> None:
        """Copies page ``src[i]`` (its first ``rows[i]`` slots, default all) to page ``dst[i]``, all layers, K and V."""
        s, d, r = _pages(src), _pages(dst), None if rows is None else _pages(rows)
        if len(s) != len(d) or (r is not None and len(r) != len(s)):
            raise ValueError("src, dst and rows must have the same length")
        _ffi.check(_ffi.lib().vfkv_pages_copy(self._h, _addr(s), _addr(d), None if r is None else _addr(r), len(s),
                                              _stream(stream)))

    def fork(self, pages: Sequence[int], kv_len: int, n_forks: int, stream=None) -> np.ndarray:
        """Page lists [n_forks, pages] of continuations of the sequence of ``kv_len`` positions in ``pages``: full pages
        are shared, a last page that is not full is copied into a page of the fork's own."""
        if not 0 <= kv_len <= _TOP or not 0 <= n_forks <= _TOP:
            raise ValueError(f"kv_len and n_forks must be between 0 and 2^32 - 1 (got {kv_len} and {n_forks})")
        used = self.pages_for(kv_len)
        p = _pages(pages)
        if len(p) < used:
            raise ValueError(f"{kv_len} positions need {used} pages, got {len(p)}")
        out = np.empty((n_forks, used), np.int32)
        _ffi.check(_ffi.lib().vfkv_pages_fork(self._h, _addr(p), kv_len, n_forks, _addr(out),
                                              _stream(stream) if self.k_ptr else None))
        return out.astype(np.int64)

    def compact(self, stream=None) -> List[int]:
        """Moves the live pages into the lowest ids; returns every page's new id (-1: the page was free)."""
        out = np.empty(self.config.n_pages, np.int32)
        _ffi.check(_ffi.lib().vfkv_pages_compact(self._h, _addr(out), _stream(stream) if self.k_ptr else None))
        return out.tolist()


def _int32(t, name: str):
    import torch
    if t.dtype is not torch.int32 or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous int32 device tensor")
    return t


class SeqBatch:
    """Sequences of one call: ``page_table`` [n_seqs, entries], ``kv_lens`` [n_seqs] (this call's tokens included) and
    ``q_offsets`` [n_seqs + 1] (None: one token per sequence), int32 device tensors.  The tensors are read when the
    work runs, so one batch object serves every step that updates them in place, captured steps too; they are kept alive."""

    def __init__(self, page_table, kv_lens, q_offsets=None, n_tokens: Optional[int] = None, max_kv_len: int = 0):
        n = kv_lens.numel()
        if page_table.dim() != 2 or page_table.shape[0] != n or kv_lens.dim() != 1:
            raise ValueError("page_table must be [n_seqs, entries] and kv_lens [n_seqs]")
        if q_offsets is not None and (q_offsets.dim() != 1 or q_offsets.numel() != n + 1):
            raise ValueError("q_offsets must be [n_seqs + 1]")
        if n_tokens is None:
            if q_offsets is not None:
                raise ValueError("n_tokens is needed with q_offsets (the offsets are on the device)")
            n_tokens = n
        if n_tokens < 0 or not 0 <= max_kv_len <= 0xFFFFFFFF:
            raise ValueError("n_tokens and max_kv_len must not be negative")
        devices = {t.device for t in (page_table, kv_lens, q_offsets) if t is not None}
        if len(devices) != 1:
            raise ValueError("page_table, kv_lens and q_offsets must be on one device")
        self.page_table, self.kv_lens = _int32(page_table, "page_table"), _int32(kv_lens, "kv_lens")
        self.q_offsets = None if q_offsets is None else _int32(q_offsets, "q_offsets")
        self.n_seqs, self.n_tokens = n, n_tokens
        self.device, self.index = kv_lens.device, kv_lens.get_device()
        self._args = _ffi.SeqBatchArgs(self.page_table.data_ptr(), self.kv_lens.data_ptr(),
                                       None if q_offsets is None else self.q_offsets.data_ptr(), n, page_table.shape[1],
                                       n_tokens, max_kv_len)
        self.args = C.byref(self._args)


class MRope:
    """Rotation of rows whose tokens have positions on one to four axes (time, height, width, ...): ``sections[a]`` pairs
    of axis ``a``, in blocks or ``interleaved``.  ``rotary_dim=0``: none."""

    def __init__(self, rotary_dim: int, freq_base: float = 10000.0, sections: Optional[Sequence[int]] = None,
                 interleaved: bool = False, rope_mode: int = _ffi.ROPE_NEOX, freq_scale: float = 1.0,
                 attn_factor: float = 1.0, eps: float = 1e-6):
        sections = [rotary_dim // 2] if sections is None else list(sections)
        if not 1 <= len(sections) <= 4:
            raise ValueError("1 to 4 axes")
        self.n_axes = len(sections)
        sections = [_fit(x) for x in sections]
        self._args = _ffi.MRopeParams(_fit(rope_mode), _fit(rotary_dim), self.n_axes, _fit(int(interleaved)),
                                      (C.c_uint32 * 4)(*(sections + [0] * (4 - self.n_axes))), freq_base, freq_scale,
                                      attn_factor, eps)
        self.args = C.byref(self._args)


class PagedWorkspace(Workspace):
    """Scratch of the paged attention calls for one cache geometry, whatever the batch."""

    def __init__(self, cache: PagedKvCache, n_heads: int):
        h = C.c_void_p()
        _ffi.check(_ffi.lib().vfkv_paged_workspace_create(cache.handle, _fit(n_heads), C.byref(h)))
        self._h = h

    @property
    def handle(self):
        return self._h


class PagedForward:
    """The calls of one model over a paged cache: its query heads, a workspace, and ``attn_scale = 1/sqrt(head_dim)``.

    Rows are [n_tokens, heads, head_dim] tensors, f32 or f16, contiguous within a token; tokens may be apart (a slice of
    one projection's output)."""

    def __init__(self, cache: PagedKvCache, n_heads: int, workspace: Optional[PagedWorkspace] = None):
        self.cache, self.n_heads, self.head_dim = cache, n_heads, cache.config.head_dim
        self.workspace = workspace or PagedWorkspace(cache, n_heads)
        self.attn_scale = 1.0 / math.sqrt(cache.config.head_dim)

    def _rows(self, t, heads: int, batch: SeqBatch, name: str):
        """(address, elements between two tokens, io dtype) of a row tensor."""
        dim = self.head_dim
        if batch.index != self.cache.device:
            raise ValueError(f"the batch is on {batch.device}, the cache on device {self.cache.device}")
        io = _IO.get(t.dtype)
        if io is None or t.get_device() != batch.index or t.shape != (batch.n_tokens, heads, dim):
            if not _IO:
                _first_use()
                return self._rows(t, heads, batch, name)
            raise ValueError(f"{name}: expected [{batch.n_tokens}, {heads}, {dim}], float32 or float16, on {batch.device}; got "
                             f"{list(t.shape)}, {t.dtype}, on {t.device}")
        token, head, elem = t.stride()
        if (elem != 1 and dim > 1) or (head != dim and heads > 1):
            raise ValueError(f"{name}: the heads of a token must be contiguous")
        if batch.n_tokens <= 1:
            token = heads * dim
        if not heads * dim <= token <= 0xFFFFFFFF:
            raise ValueError(f"{name}: tokens overlap or are too far apart (stride {token})")
        return t.data_ptr(), token, io

    def _dev(self, t, shape, dtype: str, batch: SeqBatch, name: str) -> Optional[int]:
        if t is None:
            return None
        if t.shape != shape or not t.is_contiguous() or t.get_device() != batch.index or str(t.dtype) != dtype:
            raise ValueError(f"{name}: expected a contiguous {dtype} tensor of shape {shape} on {batch.device}")
        return t.data_ptr()

    def qk_rope_kv_write(self, layer: int, batch: SeqBatch, q, k, v, rope: MRope, q_out=None, q_norm_weight=None,
                         k_norm_weight=None, positions=None, freq_factors=None, stream=None) -> None:
        """Norm (with a weight) and rotation of the query rows into ``q_out`` (default: in place) and of the key rows,
        and the append of keys and values at their tokens' positions.  ``q`` may be None.  ``positions``
        [n_axes, n_tokens] int32 (default: every axis has the token's position in its sequence)."""
        cfg = self.cache.config
        kp, ks, io = self._rows(k, cfg.n_kv_heads, batch, "k")
        vp, vs, iov = self._rows(v, cfg.n_kv_heads, batch, "v")
        qp = qs = op = os_ = None
        ioq = ioo = io
        if q is not None:
            qp, qs, ioq = self._rows(q, self.n_heads, batch, "q")
            op, os_, ioo = (qp, qs, ioq) if q_out is None else self._rows(q_out, self.n_heads, batch, "q_out")
        if not io == iov == ioq == ioo:
            raise ValueError("q, k, v and q_out must have one dtype")
        half = rope._args.rotary_dim // 2
        r = _ffi.PagedRows(qp, self._dev(q_norm_weight, (cfg.head_dim,), "torch.float32", batch, "q_norm_weight"), op, kp, vp,
                           self._dev(k_norm_weight, (cfg.head_dim,), "torch.float32", batch, "k_norm_weight"),
                           self._dev(positions, (rope.n_axes, batch.n_tokens), "torch.int32", batch, "positions"),
                           self._dev(freq_factors, (half,), "torch.float32", batch, "freq_factors"),
                           self.n_heads, io, qs or 0, os_ or 0, ks, vs)
        _ffi.check(_ffi.lib().vfkv_paged_qk_rope_kv_write(self.cache.handle, _fit(layer), batch.args, C.byref(r), rope.args,
                                                          _stream(stream, batch.index)))

    def _attention(self, fn, layer, batch, q, o, window, n_sink, scale, softcap, stream) -> None:
        if window < 0 or n_sink < 0:
            raise ValueError("window and n_sink must not be negative")
        if window > _TOP or n_sink > _TOP:                   # (every length is below 2^31: more is the same as the most)
            window, n_sink = min(window, _TOP), min(n_sink, _TOP)
        qp, qs, io = self._rows(q, self.n_heads, batch, "q")
        op, os_, ioo = self._rows(o, self.n_heads, batch, "o")
        if io != ioo:
            raise ValueError("q and o must have one dtype")
        p = _ffi.PagedAttnParams(self.n_heads, window, n_sink, io, qs, os_, self.attn_scale if scale is None else scale, softcap)
        _ffi.check(fn(self.cache.handle, _fit(layer), batch.args, C.byref(p), qp, op, self.workspace.handle, _stream(stream, batch.index)))

    def decode_attention(self, layer: int, batch: SeqBatch, q, o, window: int = 0, n_sink: int = 0,
                         scale: Optional[float] = None, softcap: float = 0.0, stream=None) -> None:
        """One token per sequence (a batch without ``q_offsets``) over the keys it sees: all, or the last ``window`` ones
        and the first ``n_sink``."""
        self._attention(_ffi.lib().vfkv_paged_decode_attention, layer, batch, q, o, window, n_sink, scale, softcap, stream)

    def prefill_attention(self, layer: int, batch: SeqBatch, q, o, window: int = 0, n_sink: int = 0,
                          scale: Optional[float] = None, softcap: float = 0.0, stream=None) -> None:
        """Causal attention of every sequence's tokens; the window is each query's own."""
        self._attention(_ffi.lib().vfkv_paged_prefill_attention, layer, batch, q, o, window, n_sink, scale, softcap, stream)
