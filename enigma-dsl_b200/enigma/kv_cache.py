"""A key/value cache in pages, shared between sequences.

`PagedKVCache` keeps the pages of every layer, a table of page numbers for each sequence
("slot"), the sequences' lengths and how many rows hold each page, all on the device.  Its
operations run on torch's current stream without reading anything back, so they can be
captured in a CUDA graph; what went wrong on the device (no free page, a slot named twice) is
kept there until `check()` raises it.  `cuda_ops.sdpa_packed` fills a cache's first tokens
with `write`, `cuda_ops.sdpa_shared_prefix` reads it (`attend`).

`QuantizedKVCache` is the same cache in 8-bit codes with a scale for each 16 tokens of a page and
head: half the bytes of bf16 to hold and to stream.  Rows are quantised as they are written, `attend`
works on the codes (`cuda_ops.sdpa_quantized`), `read` gives rows back.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

from . import _native, cuda_ops
from ._tracing import EnigmaError


class _CacheDesc(ctypes.Structure):
    """Mirror of enigma_kv_cache_desc (include/enigma_cuda.h)."""

    _fields_ = [(n, ctypes.c_int64) for n in ("layers", "pages", "heads_kv", "page", "head_dim",
                                              "elem_bytes", "slots", "table_width")] + \
               [(n, ctypes.c_void_p) for n in ("k", "v", "table", "lens", "refs", "status",
                                               "workspace")] + \
               [("workspace_bytes", ctypes.c_size_t)]


_STRIDES = struct.Struct("4q")
# enigma_kv_cache_rows (include/enigma_cuda.h): layer, entries, tokens; strides and type; pointers.
_ROWS = struct.Struct("3q")
_ROWS_KIND = struct.Struct("4q2i")
_ROWS_PTRS = struct.Struct("5Q")


class PagedKVCache:
    """k, v [layers, pages, heads_kv, page, head_dim] (bf16 or fp32) and the int32 page map:
    table [slots, width] (-1: no page), lens [slots], refs [pages]."""

    def __init__(self, k, v, table, lens, refs):
        import torch
        if k.dim() != 5 or v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("PagedKVCache: k and v must be [layers, pages, heads, page, head_dim]")
        cuda_ops._dtype_code(k)
        cuda_ops._check_cuda(k, v, table, lens, refs)
        self._setup(k, v, table, lens, refs)

    def _setup(self, k, v, table, lens, refs):
        import torch
        if any(t.dtype != torch.int32 for t in (table, lens, refs)):
            raise ValueError("PagedKVCache: table, lens and refs are int32")
        layers, pages, heads, page, head_dim = k.shape
        if table.dim() != 2 or tuple(lens.shape) != (table.shape[0],) \
                or tuple(refs.shape) != (pages,):
            raise ValueError("PagedKVCache: expected table [slots, width], lens [slots], "
                             "refs [pages]")
        self.k, self.v, self.table, self.lens, self.refs = k, v, table, lens, refs
        self.layers, self.pages, self.heads_kv, self.page, self.head_dim = k.shape
        self.slots, self.width = table.shape
        self._index, self._row = k.get_device(), (self.heads_kv, self.head_dim)
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._desc = _CacheDesc(layers, pages, heads, page, head_dim, k.element_size(),
                                self.slots, self.width, k.data_ptr(), v.data_ptr(),
                                table.data_ptr(), lens.data_ptr(), refs.data_ptr(),
                                self.status.data_ptr())
        need = ctypes.c_size_t()
        _native.call("enigma_kv_cache_workspace_bytes", ctypes.byref(self._desc),
                     ctypes.byref(need))
        self.workspace = torch.empty(need.value, dtype=torch.uint8, device=k.device)
        self._desc.workspace = self.workspace.data_ptr()
        self._desc.workspace_bytes = need.value
        self._ref = ctypes.byref(self._desc)

    @classmethod
    def empty(cls, layers: int, pages: int, page: int, heads_kv: int, head_dim: int, slots: int,
              max_len: int, dtype=None, device="cuda"):
        """A cache without tokens, for sequences of at most max_len tokens."""
        import torch
        shape = (layers, pages, heads_kv, page, head_dim)
        dtype = torch.bfloat16 if dtype is None else dtype
        width = -(-max_len // page)

        def ints(fill, *size):
            return torch.full(size, fill, dtype=torch.int32, device=device)

        return cls(torch.zeros(shape, dtype=dtype, device=device),
                   torch.zeros(shape, dtype=dtype, device=device), ints(-1, slots, width),
                   ints(0, slots), ints(0, pages))

    def _ints(self, name, values, like=None):
        """A request as an int32 device tensor (lists and host tensors are copied there)."""
        torch = cuda_ops._torch()
        if not isinstance(values, torch.Tensor):
            values = torch.as_tensor(values)
            if values.numel() == 0:
                values = values.int()
        elif values.dtype is torch.int32 and values.get_device() == self._index \
                and values.dim() == 1 and values.is_contiguous() \
                and (like is None or values.shape == like.shape):
            return values
        if values.dim() != 1:
            raise ValueError(f"{name}: expected one number per sequence")
        if like is not None and values.shape != like.shape:
            raise ValueError(f"{name}: the request's parts differ in length")
        if values.dtype != torch.int32:
            if values.dtype == torch.bool or values.is_floating_point() or values.is_complex():
                raise TypeError(f"{name}: slots, lengths and pages are whole numbers")
            # What an int32 does not hold stays out of range: refused here, or on the device.
            wide, low, high = values.long(), -1 << 31, (1 << 31) - 1
            if not wide.is_cuda and bool(((wide < low) | (wide > high)).any()):
                raise ValueError(f"{name}: a number does not fit in int32")
            values = wide.clamp(low, high).int()
        return values.to(self.k.device).contiguous()

    def _call(self, name, *args):
        cuda_ops._launch(self._index, name, self._ref, *args, cuda_ops._raw_stream(self._index))

    def fork(self, parents, children) -> None:
        """Slot children[i] continues slot parents[i]: it lets go of what it held, shares the
        parent's full pages and gets a copy of a partly filled last one."""
        parents = self._ints("fork", parents)
        children = self._ints("fork", children, parents)
        self._call("enigma_kv_cache_fork", parents.data_ptr(), children.data_ptr(),
                   parents.shape[0])

    def free(self, slots) -> None:
        """The slots let go of their pages; a page that no slot holds is free."""
        slots = self._ints("free", slots)
        self._call("enigma_kv_cache_free", slots.data_ptr(), slots.shape[0])

    def reserve(self, slots, lens) -> None:
        """Slot slots[i] grows to lens[i] tokens, taking the lowest free pages."""
        slots = self._ints("reserve", slots)
        lens = self._ints("reserve", lens, slots)
        self._call("enigma_kv_cache_reserve", slots.data_ptr(), lens.data_ptr(), slots.shape[0])

    def write(self, layer: int, new_k, new_v, slots, starts, cu) -> None:
        """Rows cu[i] .. cu[i + 1] of new_k / new_v [tokens, heads_kv, head_dim] are tokens
        starts[i], starts[i] + 1, ... of slot slots[i] in `layer` (reserved before).

        A slot may append whoever shares its pages; writing over tokens of a full page that a fork
        shares changes them for all who hold the page."""
        shape, ks, vs = new_k.shape, new_k.stride(), new_v.stride()
        if len(shape) != 3 or shape != new_v.shape or shape[1:] != self._row:
            raise ValueError(f"write: expected rows [tokens, {self._row[0]}, {self._row[1]}]")
        if new_k.dtype is not self.k.dtype or new_v.dtype is not self.k.dtype:
            raise TypeError("write: tensors must share a dtype")
        if (ks[2] != 1 or vs[2] != 1) and shape[2] > 1:
            raise ValueError("write: the last axis must be contiguous")
        cuda_ops._same_device("write", self.k, new_k, new_v)
        if not 0 <= layer < self.layers:
            raise ValueError(f"write: layer {layer} of {self.layers}")
        slots = self._ints("write", slots)
        starts = self._ints("write", starts, slots)
        cu = self._ints("write", cu)
        n = slots.shape[0]
        if cu.shape[0] != n + 1:
            raise ValueError("write: cu holds one number more than there are slots")
        self._call("enigma_kv_cache_write", layer, new_k.data_ptr(), new_v.data_ptr(),
                   _STRIDES.pack(ks[0], ks[1], vs[0], vs[1]), slots.data_ptr(),
                   starts.data_ptr(), cu.data_ptr(), n, shape[0])

    def compact(self) -> None:
        """The n pages in use take the numbers below n (rows are rewritten to match)."""
        self._call("enigma_kv_cache_compact")

    def copy_pages(self, src, dst) -> None:
        """Whole pages src[i] -> dst[i] in every layer; no page may be both."""
        src = self._ints("copy_pages", src)
        dst = self._ints("copy_pages", dst, src)
        self._call("enigma_kv_cache_copy_pages", src.data_ptr(), dst.data_ptr(), src.numel())

    def attend(self, layer: int, q, slots=None, prefix_len: int = 0,
               scale: Optional[float] = None, out=None, workspace=None):
        """cuda_ops.sdpa_shared_prefix over one layer of this cache."""
        return cuda_ops.sdpa_shared_prefix(q, self.k[layer], self.v[layer], self.table, self.lens,
                                           prefix_len=prefix_len,
                                           slots=None if slots is None
                                           else self._ints("attend", slots),
                                           scale=scale, out=out, workspace=workspace)

    def check(self) -> None:
        """Waits for the device and raises if a request since the last check was not met."""
        cuda_ops._torch().cuda.synchronize(self._index)   # requests may run on any stream
        code = int(self.status.item())
        if code:
            self.status.zero_()
        if code & _native.CACHE_SHARED:
            raise EnigmaError("paged cache: a write named a page that forks share")
        if code & _native.CACHE_BAD_REQUEST:
            raise EnigmaError("paged cache: a request named a slot or page that does not exist, "
                              "a slot twice, a parent as its child, or a length that does not "
                              "fit its row")
        if code & _native.CACHE_FULL:
            raise EnigmaError("paged cache: not enough free pages")


class _QuantizedDesc(ctypes.Structure):
    """Mirror of enigma_kv_cache_q8_desc (include/enigma_cuda.h)."""

    _fields_ = [("cache", _CacheDesc), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
                ("code", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class QuantizedKVCache(PagedKVCache):
    """A paged cache in 8-bit codes: k, v [layers, pages, heads_kv, page, head_dim] int8 or
    float8_e4m3fn, k_scale, v_scale [layers, pages, heads_kv, page / 16] fp32; a code x stands for
    x * scale.  The page map and its operations are PagedKVCache's, pages move with their scales.

    A scale is the least power of two that brings its block's largest magnitude to at most 127
    (int8) or 448 (e4m3).  Appending to a partly filled block may raise its scale; its earlier tokens
    are then rounded once more, and stay within one step of what was written, however often."""

    def __init__(self, k, v, k_scale, v_scale, table, lens, refs):
        import torch
        if k.dim() != 5 or v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("QuantizedKVCache: k and v must be [layers, pages, heads, page, head_dim]")
        code = cuda_ops._code_of(k.dtype)
        cuda_ops._check_cuda(k, v, k_scale, v_scale, table, lens, refs)
        layers, pages, heads, page, head_dim = k.shape
        if page not in (16, 32, 64, 128) or head_dim % 16 or not 0 < head_dim <= 256:
            raise ValueError("QuantizedKVCache: page must be 16, 32, 64 or 128, head_dim a multiple "
                             "of 16 up to 256")
        scales = (layers, pages, heads, page // _native.SCALE_BLOCK)
        if any(tuple(x.shape) != scales or x.dtype != torch.float32 for x in (k_scale, v_scale)):
            raise ValueError("QuantizedKVCache: scales are fp32 [layers, pages, heads, page / "
                             f"{_native.SCALE_BLOCK}]")
        if k.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError("QuantizedKVCache: k and v must be 16-byte aligned")
        self.k_scale, self.v_scale = k_scale, v_scale
        self._setup(k, v, table, lens, refs)
        self._q8 = _QuantizedDesc(self._desc, k_scale.data_ptr(), v_scale.data_ptr(), code, 0)
        self._q8_ref = ctypes.byref(self._q8)
        self._heads = {}         # checked calls' sizes, strides and types

    @classmethod
    def empty(cls, layers: int, pages: int, page: int, heads_kv: int, head_dim: int, slots: int,
              max_len: int, dtype=None, device="cuda"):
        """A cache without tokens, for sequences of at most max_len tokens; dtype (of the codes):
        torch.int8 (the default) or torch.float8_e4m3fn."""
        import torch
        dtype = torch.int8 if dtype is None else dtype
        cuda_ops._code_of(dtype)
        shape = (layers, pages, heads_kv, page, head_dim)
        scales = (layers, pages, heads_kv, page // _native.SCALE_BLOCK)

        def ints(fill, *size):
            return torch.full(size, fill, dtype=torch.int32, device=device)

        codes = [torch.zeros(shape, dtype=torch.int8, device=device).view(dtype) for _ in range(2)]
        return cls(*codes, *(torch.zeros(scales, device=device) for _ in range(2)),
                   ints(-1, slots, -(-max_len // page)), ints(0, slots), ints(0, pages))

    def _call_q8(self, name, *args):
        cuda_ops._launch(self._index, name, self._q8_ref, *args, cuda_ops._raw_stream(self._index))

    def fork(self, parents, children) -> None:
        parents = self._ints("fork", parents)
        children = self._ints("fork", children, parents)
        self._call_q8("enigma_kv_cache_q8_fork", parents.data_ptr(), children.data_ptr(),
                      parents.shape[0])

    def compact(self) -> None:
        self._call_q8("enigma_kv_cache_q8_compact")

    def copy_pages(self, src, dst) -> None:
        src = self._ints("copy_pages", src)
        dst = self._ints("copy_pages", dst, src)
        self._call_q8("enigma_kv_cache_q8_copy_pages", src.data_ptr(), dst.data_ptr(), src.numel())

    fork.__doc__ = PagedKVCache.fork.__doc__
    compact.__doc__ = PagedKVCache.compact.__doc__
    copy_pages.__doc__ = PagedKVCache.copy_pages.__doc__

    def _checked(self, key, check):
        """What `check(*key)` packs, made once for these sizes, strides and types."""
        head = self._heads.get(key)
        if head is None:
            head = check(*key)
            if len(self._heads) >= 256:
                self._heads.clear()
            self._heads[key] = head
        return head

    def _rows_head(self, name, layer, k, v):
        """Checks the (shape, stride, dtype) of a write's or read's rows; strides and type, their number."""
        (shape, ks, kind), vs = k, v[1]
        if len(shape) != 3 or shape != v[0] or shape[1:] != self._row:
            raise ValueError(f"{name}: expected rows [tokens, {self._row[0]}, {self._row[1]}]")
        dtype = cuda_ops._check_rows(name, kind, k, v)
        if name == "read":
            cuda_ops._check_distinct(name, k, v)
        if not 0 <= layer < self.layers:
            raise ValueError(f"{name}: layer {layer} of {self.layers}")
        return _ROWS_KIND.pack(ks[0], ks[1], vs[0], vs[1], dtype, 0), shape[0]

    def _rows_call(self, name, entry, layer, k, v, slots, starts, cu):
        kind, tokens = self._checked(
            (name, layer, (k.shape, k.stride(), k.dtype), (v.shape, v.stride(), v.dtype)),
            self._rows_head)
        cuda_ops._same_device(name, self.k, k, v)
        if not self._are_ints(slots, starts, cu):
            slots = self._ints(name, slots)
            starts = self._ints(name, starts)
            cu = self._ints(name, cu)
        n = slots.shape[0]
        if starts.shape[0] != n:
            raise ValueError(f"{name}: the request's parts differ in length")
        if cu.shape[0] != n + 1:
            raise ValueError(f"{name}: cu holds one number more than there are slots")
        self._call_q8(entry, _ROWS.pack(layer, n, tokens) + kind + _ROWS_PTRS.pack(
            k.data_ptr(), v.data_ptr(), slots.data_ptr(), starts.data_ptr(), cu.data_ptr()))

    def _are_ints(self, *parts) -> bool:
        """Whether a request's parts are what `_ints` would make of them."""
        int32, index = cuda_ops._torch().int32, self._index
        try:
            for x in parts:
                if x.dtype is not int32 or x.get_device() != index or x.dim() != 1 \
                        or not x.is_contiguous():
                    return False
        except (AttributeError, TypeError):                  # a list, an array
            return False
        return True

    def write(self, layer: int, new_k, new_v, slots, starts, cu) -> None:
        """Rows cu[i] .. cu[i + 1] of new_k / new_v [tokens, heads_kv, head_dim], bf16 or fp32, are
        tokens starts[i], starts[i] + 1, ... of slot slots[i] in `layer` (reserved before).

        A slot's tokens are written in order; going back to an earlier token is fine and cuts off
        what the block of 16 held behind.  Pages that forks share are not written (`check` says so;
        appending never meets one), nor is a block that two entries of one call name.  A value that is
        not finite makes its block of 16 tokens NaN."""
        self._rows_call("write", "enigma_kv_cache_q8_write", layer, new_k, new_v, slots, starts, cu)

    def read(self, layer: int, slots, starts, cu, tokens: Optional[int] = None, dtype=None,
             out_k=None, out_v=None):
        """Tokens starts[i], starts[i] + 1, ... of slot slots[i] in `layer` as rows cu[i] .. cu[i + 1]
        of k, v [tokens, heads_kv, head_dim], e.g. earlier context for `cuda_ops.sdpa_packed`.

        tokens: the number of rows, by default cu's last number (which must then be on the host);
        dtype bf16 (the default; it holds every code times a power of two) or fp32; out_k / out_v:
        tensors to write instead.  A token that the slot does not hold gives zeros; rows that no entry
        names are not written (they stay what they were in out_k and out_v)."""
        import torch
        if (out_k is None) != (out_v is None):
            raise ValueError("read: out_k and out_v come together")
        if out_k is None:
            if tokens is None:
                if isinstance(cu, torch.Tensor) and cu.is_cuda:
                    raise ValueError("read: tokens must be given where cu is on the device")
                tokens = int(cu[-1]) if len(cu) else 0
            dtype = torch.bfloat16 if dtype is None else dtype
            device = self.k.device
            out_k = torch.empty(int(tokens), *self._row, dtype=dtype, device=device)
            out_v = torch.empty(int(tokens), *self._row, dtype=dtype, device=device)
        elif tokens not in (None, out_k.shape[0]) or dtype not in (None, out_k.dtype):
            raise ValueError("read: out_k and out_v have another size or type")
        self._rows_call("read", "enigma_kv_cache_q8_read", layer, out_k, out_v, slots, starts, cu)
        return out_k, out_v

    def attend(self, layer: int, q, slots=None, *, scale: Optional[float] = None, out=None,
               workspace=None):
        """cuda_ops.sdpa_quantized over one layer of this cache.  Every sequence reads its keys for
        itself: there is no prefix_len, which PagedKVCache.attend takes after slots, so what follows
        slots is named."""
        slots = None if slots is None else self._ints("attend", slots)
        head, need, pages = self._checked(
            (layer, (q.shape, q.stride(), q.dtype), None if slots is None else slots.shape,
             None if out is None else (out.shape, out.stride(), out.dtype), scale), self._attend_head)
        return cuda_ops._sdpa_quantized(self._index, head, need, pages, q, slots, out, workspace)

    def _attend_head(self, layer, q, slots, out, scale):
        """Checks the (shape, stride, dtype) of an attend; the desc's head, bytes of workspace, and the
        addresses of the layer's pages, scales, the table and the lengths."""
        if not 0 <= layer < self.layers:
            raise ValueError(f"attend: layer {layer} of {self.layers}")
        pools = (self.k, self.v, self.k_scale, self.v_scale)
        described = [(x.shape, x.stride(), x.dtype)
                     for x in [y[layer] for y in pools] + [self.table, self.lens]]
        head, need = cuda_ops._quantized_head(
            self._index, q, *described, None if slots is None else (slots, (1,), self.table.dtype),
            out, scale)
        return head, need, (*(x.data_ptr() + layer * x.stride(0) * x.element_size() for x in pools),
                            self.table.data_ptr(), self.lens.data_ptr())
