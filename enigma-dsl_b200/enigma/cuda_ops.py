"""torch-tensor front end of the sm_100a operators.

PyTorch only provides device memory and the current stream here; all compute
is in libenigma_cuda.so.  Every function launches asynchronously on the
current torch stream of the tensors' device and returns the output tensor.
Inputs must be contiguous CUDA tensors; there is no CPU path.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import Optional

from . import _native

_initialised: set = set()


_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch  # on first use: the package imports without torch for host-only use
        _torch_module = torch
    return _torch_module


def ensure_device(device_index: int) -> None:
    if device_index not in _initialised:
        _native.call("enigma_init", device_index)
        _initialised.add(device_index)


def _stream_ptr(t) -> int:
    torch = _torch()
    return torch.cuda.current_stream(t.device).cuda_stream


def _check_cuda(*ts):
    dev = None
    for t in ts:
        if not t.is_cuda:
            raise ValueError("enigma CUDA operators take CUDA tensors (no CPU fallback)")
        if not t.is_contiguous():
            raise ValueError("enigma CUDA operators take contiguous tensors")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError("all tensors must be on the same device")
    ensure_device(dev.index if dev.index is not None else 0)


def _dtype_code(t) -> int:
    torch = _torch()
    if t.dtype == torch.float32:
        return _native.DTYPE_F32
    if t.dtype == torch.bfloat16:
        return _native.DTYPE_BF16
    raise TypeError(f"unsupported dtype {t.dtype}: expected float32 or bfloat16")


def rmsnorm(x, w, eps: float = 1e-6, out=None):
    """y = x * rsqrt(mean(x^2, -1) + eps) * w over the last axis (fp32 accumulate)."""
    torch = _torch()
    if out is None:
        out = torch.empty_like(x)
    _check_cuda(x, w, out)
    hidden = x.shape[-1]
    if w.numel() != hidden or w.dtype != x.dtype or out.dtype != x.dtype:
        raise ValueError("rmsnorm: w must have hidden elements and x's dtype")
    rows = x.numel() // hidden if hidden else 0
    _native.call("enigma_rmsnorm", _dtype_code(x), x.data_ptr(), w.data_ptr(), out.data_ptr(),
                 rows, hidden, ctypes.c_float(eps), _stream_ptr(x))
    return out


def gemm(a, b, out=None, accumulate: bool = False):
    """C = A @ B for row-major A [M,K], B [K,N]; bf16 (tensor cores) or fp32 (CUDA cores).

    accumulate=True computes C += A @ B and is fp32-only (the reference's gemm_k4).
    """
    torch = _torch()
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[0]:
        raise ValueError(f"gemm: shapes {tuple(a.shape)} x {tuple(b.shape)} do not chain")
    if a.dtype != b.dtype:
        raise TypeError("gemm: A and B must share a dtype")
    m, k = a.shape
    n = b.shape[1]
    if out is None:
        if accumulate:
            raise ValueError("gemm: accumulate=True needs out")
        out = torch.empty((m, n), dtype=a.dtype, device=a.device)
    _check_cuda(a, b, out)
    if a.dtype == torch.bfloat16:
        if accumulate:
            raise TypeError("gemm: accumulate is fp32-only")
        _native.call("enigma_gemm_bf16", a.data_ptr(), b.data_ptr(), out.data_ptr(), m, n, k,
                     _stream_ptr(a))
    elif a.dtype == torch.float32:
        _native.call("enigma_gemm_f32", a.data_ptr(), b.data_ptr(), out.data_ptr(), m, n, k,
                     int(accumulate), _stream_ptr(a))
    else:
        raise TypeError(f"gemm: unsupported dtype {a.dtype}")
    return out


def sdpa(q, k, v, scale: Optional[float] = None, causal: bool = False, out=None):
    """O = softmax(scale * Q K^T [causal]) V for [B, H, S, D] tensors (GQA when Hk < Hq).

    scale defaults to 1/sqrt(D).  causal keeps key j <= i + (Sk - Sq).
    """
    torch = _torch()
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("sdpa: expected [B, H, S, D] tensors")
    b, hq, sq, d = q.shape
    bk, hk, sk, dk = k.shape
    if bk != b or dk != d or tuple(v.shape) != tuple(k.shape):
        raise ValueError("sdpa: K/V shapes do not match Q")
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.empty_like(q)
    _check_cuda(q, k, v, out)
    fn = "enigma_sdpa_bf16" if q.dtype == torch.bfloat16 else "enigma_sdpa_f32"
    if q.dtype not in (torch.bfloat16, torch.float32) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("sdpa: Q/K/V must all be bf16 or all fp32")
    _native.call(fn, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), b, hq, hk, sq, sk,
                 d, ctypes.c_float(scale), int(causal), _stream_ptr(q))
    return out


class PackedPlan:
    """The work list of `sdpa_packed` for prompts of these lengths, made once per batch.

    lens_q / lens_k: tokens of each sequence's queries and keys (lens_k defaults to lens_q; a
    sequence with more keys than queries continues an earlier part of its context).
    """

    def __init__(self, lens_q, lens_k=None, *, heads_q: int, heads_kv: int, causal: bool = True,
                 device="cuda"):
        torch = _torch()
        lens_q = [int(n) for n in lens_q]
        lens_k = lens_q if lens_k is None else [int(n) for n in lens_k]
        if len(lens_q) != len(lens_k):
            raise ValueError("PackedPlan: lens_q and lens_k differ in number")
        n = len(lens_q)
        c_q, c_k = (ctypes.c_int64 * n)(*lens_q), (ctypes.c_int64 * n)(*lens_k)
        count = ctypes.c_int64()
        args = (c_q, c_k, n, heads_q, heads_kv, int(causal))
        _native.call("enigma_sdpa_packed_plan", *args, None, 0, ctypes.byref(count))
        ints = torch.empty(count.value, dtype=torch.int32)
        _native.call("enigma_sdpa_packed_plan", *args,
                     ctypes.cast(ints.data_ptr(), ctypes.POINTER(ctypes.c_int32)), count.value,
                     ctypes.byref(count))
        self.heads_q, self.heads_kv, self.causal = int(heads_q), int(heads_kv), bool(causal)
        self.tokens_q, self.tokens_k = sum(lens_q), sum(lens_k)
        self.header = tuple(ints[:_native.PACKED_PLAN_HEADER].tolist())
        self.ints = ints.to(device)
        self._workspace = {}

    def workspace_bytes(self, head_dim: int) -> int:
        """Device memory that a call with this plan needs (0 unless it splits rows)."""
        if head_dim not in self._workspace:
            need = ctypes.c_size_t()
            _native.call("enigma_sdpa_packed_workspace_bytes",
                         (ctypes.c_int32 * len(self.header))(*self.header), head_dim,
                         ctypes.byref(need))
            self._workspace[head_dim] = need.value
        return self._workspace[head_dim]


# enigma_sdpa_packed_desc (include/enigma_cuda.h): sizes and strides, scale and flags, the plan's
# header, pointers.  Packed bytes cost a third of filling a ctypes structure.
_PACKED_DESC = struct.Struct(f"13qf3i{_native.PACKED_PLAN_HEADER}i8Q")


_CUDA = "cuda"


def _raw_stream(t) -> int:
    """The current stream of t's device, without the Stream object that _stream_ptr makes."""
    return _torch()._C._cuda_getCurrentRawStream(t.device.index)


def _check_rows(name, *ts):
    """CUDA tensors of one device and dtype whose last axis is contiguous; the dtype's code."""
    first = ts[0]
    device, dtype = first.device, first.dtype
    if device.type != _CUDA:
        raise ValueError("enigma CUDA operators take CUDA tensors (no CPU fallback)")
    for t in ts:
        if t.device != device:
            raise ValueError("enigma CUDA operators take CUDA tensors of one device")
        if t.dtype != dtype:
            raise TypeError(f"{name}: tensors must share a dtype")
        if t.stride(-1) != 1 and t.shape[-1] > 1:
            raise ValueError(f"{name}: the last axis must be contiguous")
    if device.index not in _initialised:
        ensure_device(device.index)
    return _dtype_code(first)


def _scratch(name, workspace, need, like):
    """(address, bytes) of the caller's workspace or of a new one, and what keeps it alive."""
    if workspace is None:
        if need == 0:
            return 0, 0, None
        workspace = like.new_empty(need, dtype=_torch().uint8)
        return workspace.data_ptr(), need, workspace
    if workspace.device != like.device or not workspace.is_contiguous():
        raise ValueError(f"{name}: workspace must be contiguous on the data's device")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace


def sdpa_packed(q, k, v, plan: PackedPlan, scale: Optional[float] = None, out=None,
                return_lse: bool = False, workspace=None):
    """Attention over whole prompts packed one after the other.

    q [tokens_q, Hq, D], k / v [tokens_k, Hkv, D] (GQA when Hkv < Hq), any token and head
    strides, e.g. slices of one fused projection's output.  Row i of a sequence sees its keys
    j <= i + len_k - len_q (all of them with a plan made with causal=False); a row that sees
    none is zero.  scale defaults to 1/sqrt(D).  workspace: a uint8 tensor of
    plan.workspace_bytes(D) bytes to use instead of an allocation per call.  Returns out
    [tokens_q, Hq, D], and with return_lse the fp32 log-sum-exp [tokens_q, Hq] too.
    """
    torch = _torch()
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("sdpa_packed: expected [tokens, heads, head_dim] tensors")
    tq, hq, d = q.shape
    tk, hk, dk = k.shape
    if dk != d or v.shape != k.shape:
        raise ValueError("sdpa_packed: K/V shapes do not match Q")
    if (hq, hk) != (plan.heads_q, plan.heads_kv):
        raise ValueError("sdpa_packed: the plan was made for other heads")
    if (tq, tk) != (plan.tokens_q, plan.tokens_k):
        raise ValueError(f"sdpa_packed: the plan's lengths sum to {plan.tokens_q} / "
                         f"{plan.tokens_k} tokens, the tensors hold {tq} / {tk}")
    if out is None:
        dtype = _check_rows("sdpa_packed", q, k, v)
        out = q.new_empty((tq, hq, d))
    elif out.shape != q.shape:
        raise ValueError("sdpa_packed: out must have q's shape")
    else:
        dtype = _check_rows("sdpa_packed", q, k, v, out)
    if plan.ints.device != q.device:
        raise ValueError("sdpa_packed: the plan is on another device")
    lse = q.new_empty((tq, hq), dtype=torch.float32) if return_lse else None
    ws, ws_bytes, keep = _scratch("sdpa_packed", workspace, plan.workspace_bytes(d), q)
    qs, ks, vs, os = q.stride(), k.stride(), v.stride(), out.stride()
    desc = _PACKED_DESC.pack(tq, tk, hq, hk, d, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0],
                             os[1], 1.0 / math.sqrt(d) if scale is None else scale, plan.causal,
                             dtype, 0, *plan.header, plan.ints.data_ptr(), q.data_ptr(),
                             k.data_ptr(), v.data_ptr(), out.data_ptr(),
                             lse.data_ptr() if return_lse else 0, ws, ws_bytes)
    _native.call("enigma_sdpa_packed", desc, _raw_stream(q))
    return (out, lse) if return_lse else out


# enigma_sdpa_shared_prefix_desc: sizes and strides, scale and dtype, pointers, workspace.
_SHARED_DESC = struct.Struct("15qfi9Q")


@functools.lru_cache(maxsize=4096)
def _shared_workspace_bytes(device_index, *sizes) -> int:
    """enigma_sdpa_shared_prefix_workspace_bytes for the desc's sizes (it reads nothing else)."""
    need = ctypes.c_size_t()
    _native.call("enigma_sdpa_shared_prefix_workspace_bytes",
                 _SHARED_DESC.pack(*sizes[:9], 0, 0, 0, 0, 0, 0, 1.0, sizes[9], *([0] * 9)),
                 ctypes.byref(need))
    return need.value


def _check_int32(name, device, *ts):
    int32 = _torch().int32
    for t in ts:
        if t.dtype != int32 or t.device != device or not t.is_contiguous():
            raise ValueError(f"{name}: tables, lengths and slots are contiguous int32 tensors on "
                             f"the data's device")


def sdpa_shared_prefix(q, k_pages, v_pages, table, lens, prefix_len: int = 0, slots=None,
                       scale: Optional[float] = None, out=None, workspace=None):
    """One new token per sequence over a paged cache whose sequences share their first tokens.

    q [B, Hq, D]; k_pages / v_pages [pages, Hkv, page, D] (one layer of a cache); table
    [n, width] int32 page numbers, lens [n] int32; sequence b uses row slots[b] (default: row
    b).  Sequence b attends to its first lens keys; those below prefix_len are the same for
    the whole batch and are read once for all, through sequence 0's row.  A sequence without
    keys gives zeros.  workspace: a uint8 tensor to use instead of an allocation per call
    (as many bytes as enigma_sdpa_shared_prefix_workspace_bytes says).  Returns out [B, Hq, D].
    """
    torch = _torch()
    if q.dim() != 3 or k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
        raise ValueError("sdpa_shared_prefix: expected q [B, Hq, D] and pages [P, Hkv, page, D]")
    b, hq, d = q.shape
    pages, hk, page, dk = k_pages.shape
    if dk != d:
        raise ValueError("sdpa_shared_prefix: K/V head_dim does not match Q")
    if table.dim() != 2 or lens.dim() != 1 or lens.shape[0] != table.shape[0]:
        raise ValueError("sdpa_shared_prefix: expected table [n, width] and lens [n]")
    if slots is not None and tuple(slots.shape) != (b,):
        raise ValueError("sdpa_shared_prefix: slots must name one row per sequence")
    if out is None:
        dtype = _check_rows("sdpa_shared_prefix", q, k_pages, v_pages)
        out = q.new_empty((b, hq, d))
    elif out.shape != q.shape:
        raise ValueError("sdpa_shared_prefix: out must have q's shape")
    else:
        dtype = _check_rows("sdpa_shared_prefix", q, k_pages, v_pages, out)
    ks, vs = k_pages.stride(), v_pages.stride()
    if ks[1:] != (page * d, d, 1) or vs[1:] != (page * d, d, 1):
        raise ValueError("sdpa_shared_prefix: a page must be contiguous")
    _check_int32("sdpa_shared_prefix", q.device, table, lens, *(() if slots is None else (slots,)))
    sizes = (b, hq, hk, d, page, pages, table.shape[1], table.shape[0], int(prefix_len))
    need = _shared_workspace_bytes(q.device.index, *sizes, dtype)
    ws, ws_bytes, keep = _scratch("sdpa_shared_prefix", workspace, need, q)
    qs, os = q.stride(), out.stride()
    desc = _SHARED_DESC.pack(*sizes, qs[0], qs[1], os[0], os[1], ks[0], vs[0],
                             1.0 / math.sqrt(d) if scale is None else scale, dtype,
                             table.data_ptr(), lens.data_ptr(),
                             0 if slots is None else slots.data_ptr(), q.data_ptr(),
                             k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), ws, ws_bytes)
    _native.call("enigma_sdpa_shared_prefix", desc, _raw_stream(q))
    return out


def synchronize(device_index: int = 0) -> None:
    """Synchronize the device and raise if a kernel reported a device-side timeout."""
    ensure_device(device_index)
    _native.call("enigma_synchronize", None)
