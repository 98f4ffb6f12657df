"""A key/value cache in pages, shared between sequences.

`PagedKVCache` keeps the pages of every layer, a table of page numbers for each sequence
("slot"), the sequences' lengths and how many rows hold each page, all on the device.  Its
operations run on torch's current stream without reading anything back, so they can be
captured in a CUDA graph; what went wrong on the device (no free page, a slot named twice) is
kept there until `check()` raises it.  `cuda_ops.sdpa_packed` fills a cache's first tokens
with `write`, `cuda_ops.sdpa_shared_prefix` reads it (`attend`).
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


class PagedKVCache:
    """k, v [layers, pages, heads_kv, page, head_dim] (bf16 or fp32) and the int32 page map:
    table [slots, width] (-1: no page), lens [slots], refs [pages]."""

    def __init__(self, k, v, table, lens, refs):
        import torch
        if k.dim() != 5 or v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("PagedKVCache: k and v must be [layers, pages, heads, page, head_dim]")
        cuda_ops._dtype_code(k)
        cuda_ops._check_cuda(k, v, table, lens, refs)
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
        if code & _native.CACHE_BAD_REQUEST:
            raise EnigmaError("paged cache: a request named a slot or page that does not exist, "
                              "a slot twice, a parent as its child, or a length that does not "
                              "fit its row")
        if code & _native.CACHE_FULL:
            raise EnigmaError("paged cache: not enough free pages")
