"""torch-tensor front end of the sm_100a operators.

PyTorch only provides device memory and the current stream here; all compute
is in libenigma_cuda.so.  Every function launches asynchronously on the
current torch stream of the tensors' device and returns the output tensor.
Inputs must be contiguous CUDA tensors; there is no CPU path.
"""
from __future__ import annotations

import contextlib
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
    """Checks and prepares a device on first use; the caller's current device stays current."""
    if device_index not in _initialised:
        with _torch().cuda.device(device_index):
            _native.call("enigma_init", device_index)
        _initialised.add(device_index)


def _launch(index: int, name: str, *args) -> None:
    """Calls C entry `name` with device `index` current (the library launches on the current device,
    whose streams, SM count and status word it takes), and raises if it fails."""
    torch = _torch()
    if torch._C._cuda_getDevice() == index:
        status = getattr(_native.lib(), name)(*args)
    else:
        with torch.cuda.device(index):
            status = getattr(_native.lib(), name)(*args)
    if status:
        _native.check(status, name)


def _current(device):
    """A context in which `device` is current, where it names a CUDA device by its number."""
    torch = _torch()
    device = torch.device(device)
    if device.type != "cuda" or device.index is None:
        return contextlib.nullcontext()
    return torch.cuda.device(device.index)


def _stream_ptr(t) -> int:
    torch = _torch()
    return torch.cuda.current_stream(t.device).cuda_stream


def _check_cuda(*ts) -> int:
    """Index of the CUDA device that all tensors are on, contiguous."""
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
    index = ts[0].get_device()
    ensure_device(index)
    return index


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
    index = _check_cuda(x, w, out)
    hidden = x.shape[-1]
    if w.numel() != hidden or w.dtype != x.dtype or out.dtype != x.dtype:
        raise ValueError("rmsnorm: w must have hidden elements and x's dtype")
    rows = x.numel() // hidden if hidden else 0
    _launch(index, "enigma_rmsnorm", _dtype_code(x), x.data_ptr(), w.data_ptr(), out.data_ptr(),
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
    index = _check_cuda(a, b, out)
    if a.dtype == torch.bfloat16:
        if accumulate:
            raise TypeError("gemm: accumulate is fp32-only")
        _launch(index, "enigma_gemm_bf16", a.data_ptr(), b.data_ptr(), out.data_ptr(), m, n, k,
                _stream_ptr(a))
    elif a.dtype == torch.float32:
        _launch(index, "enigma_gemm_f32", a.data_ptr(), b.data_ptr(), out.data_ptr(), m, n, k,
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
    index = _check_cuda(q, k, v, out)
    fn = "enigma_sdpa_bf16" if q.dtype == torch.bfloat16 else "enigma_sdpa_f32"
    if q.dtype not in (torch.bfloat16, torch.float32) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("sdpa: Q/K/V must all be bf16 or all fp32")
    _launch(index, fn, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), b, hq, hk, sq, sk,
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
        # The work is dealt out over the SMs of the plan's device (on the host: as many as a B200 has).
        with _current(device):
            _native.call("enigma_sdpa_packed_plan", *args, None, 0, ctypes.byref(count))
            ints = torch.empty(count.value, dtype=torch.int32)
            _native.call("enigma_sdpa_packed_plan", *args,
                         ctypes.cast(ints.data_ptr(), ctypes.POINTER(ctypes.c_int32)), count.value,
                         ctypes.byref(count))
        self.heads_q, self.heads_kv, self.causal = int(heads_q), int(heads_kv), bool(causal)
        self.tokens_q, self.tokens_k = sum(lens_q), sum(lens_k)
        self.header = tuple(ints[:_native.PACKED_PLAN_HEADER].tolist())
        self.ints = ints.to(device)
        self.heads = {}          # checked calls' sizes, strides and types

    def workspace_bytes(self, head_dim: int) -> int:
        """Device memory that a call with this plan needs (0 unless it splits rows)."""
        need = ctypes.c_size_t()
        _native.call("enigma_sdpa_packed_workspace_bytes",
                     (ctypes.c_int32 * len(self.header))(*self.header), head_dim,
                     ctypes.byref(need))
        return need.value


# The serving operators are called for every layer and token, on calls of a few microseconds: what
# depends on sizes, strides and types alone is checked and packed once per combination.
#
# enigma_sdpa_packed_desc (include/enigma_cuda.h): sizes and strides, scale and flags, the plan's
# header; then pointers.
_PACKED_HEAD = struct.Struct(f"13qf3i{_native.PACKED_PLAN_HEADER}i")
_PACKED_PTRS = struct.Struct("8Q")
# enigma_sdpa_shared_prefix_desc: sizes and strides, scale and dtype; then pointers.
_SHARED_HEAD = struct.Struct("15qfi")
_SHARED_PTRS = struct.Struct("9Q")


def _raw_stream(index: int) -> int:
    """The current stream of device `index`, without the Stream object that _stream_ptr makes."""
    return _torch()._C._cuda_getCurrentRawStream(index)


def _same_device(name, first, *others) -> int:
    """Index of the CUDA device that all tensors are on."""
    index = first.get_device()
    if index < 0:
        raise ValueError("enigma CUDA operators take CUDA tensors (no CPU fallback)")
    for t in others:
        if t.get_device() != index:
            raise ValueError(f"{name}: all tensors must be on the same device")
    if index not in _initialised:
        ensure_device(index)
    return index


def _check_rows(name, dtype, *tensors):
    """(shape, stride, dtype) of tensors: one dtype, a contiguous last axis.  The dtype's code."""
    torch = _torch()
    for shape, stride, other in tensors:
        if other != dtype:
            raise TypeError(f"{name}: tensors must share a dtype")
        if stride[-1] != 1 and shape[-1] > 1:
            raise ValueError(f"{name}: the last axis must be contiguous")
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"unsupported dtype {dtype}: expected float32 or bfloat16")
    return _native.DTYPE_F32 if dtype == torch.float32 else _native.DTYPE_BF16


def _dense(shape, stride) -> bool:
    """Whether the elements lie one after the other; axes of length 1 may have any stride."""
    step = 1
    for n, s in zip(reversed(shape), reversed(stride)):
        if n > 1 and s != step:
            return 0 in shape
        step *= n
    return True


def _contiguous_like(q):
    """An uninitialised contiguous tensor of q's shape (new_empty takes a microsecond longer)."""
    torch = _torch()
    return torch.empty_like(q, memory_format=torch.contiguous_format)


def _scratch(name, workspace, need, like):
    """(address, bytes) of the caller's workspace or of a new one, and what keeps it alive."""
    if workspace is None:
        if need == 0:
            return 0, 0, None
        workspace = like.new_empty(need, dtype=_torch().uint8)
        return workspace.data_ptr(), need, workspace
    if workspace.get_device() != like.get_device() or not workspace.is_contiguous():
        raise ValueError(f"{name}: workspace must be contiguous on the data's device")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace


def _packed_head(plan, q, k, v, out, scale):
    """Checks the (shape, stride, dtype) of a call with this plan and packs the desc's head."""
    if len(q[0]) != 3 or len(k[0]) != 3 or len(v[0]) != 3:
        raise ValueError("sdpa_packed: expected [tokens, heads, head_dim] tensors")
    tq, hq, d = q[0]
    tk, hk, dk = k[0]
    if dk != d or v[0] != k[0]:
        raise ValueError("sdpa_packed: K/V shapes do not match Q")
    if (hq, hk) != (plan.heads_q, plan.heads_kv):
        raise ValueError("sdpa_packed: the plan was made for other heads")
    if (tq, tk) != (plan.tokens_q, plan.tokens_k):
        raise ValueError(f"sdpa_packed: the plan's lengths sum to {plan.tokens_q} / "
                         f"{plan.tokens_k} tokens, the tensors hold {tq} / {tk}")
    if out is None:
        out = (q[0], (hq * d, d, 1), q[2])
    elif out[0] != q[0]:
        raise ValueError("sdpa_packed: out must have q's shape")
    dtype = _check_rows("sdpa_packed", q[2], q, k, v, out)
    return (_PACKED_HEAD.pack(tq, tk, hq, hk, d, *q[1][:2], *k[1][:2], *v[1][:2], *out[1][:2],
                              1.0 / math.sqrt(d) if scale is None else scale, plan.causal, dtype,
                              0, *plan.header), plan.workspace_bytes(d))


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
    key = ((q.shape, q.stride(), q.dtype), (k.shape, k.stride(), k.dtype),
           (v.shape, v.stride(), v.dtype),
           None if out is None else (out.shape, out.stride(), out.dtype), scale)
    head = plan.heads.get(key)
    if head is None:
        head = _packed_head(plan, *key)
        if len(plan.heads) >= 64:
            plan.heads.clear()
        plan.heads[key] = head
    if out is None:
        out = _contiguous_like(q)
        index = _same_device("sdpa_packed", q, k, v, plan.ints)
    else:
        index = _same_device("sdpa_packed", q, k, v, plan.ints, out)
    lse = q.new_empty(q.shape[:2], dtype=_torch().float32) if return_lse else None
    ws, ws_bytes, keep = _scratch("sdpa_packed", workspace, head[1], q)
    desc = head[0] + _PACKED_PTRS.pack(plan.ints.data_ptr(), q.data_ptr(), k.data_ptr(),
                                       v.data_ptr(), out.data_ptr(),
                                       lse.data_ptr() if return_lse else 0, ws, ws_bytes)
    _launch(index, "enigma_sdpa_packed", desc, _raw_stream(index))
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=1024)
def _shared_head(index, q, k, v, table, lens, slots, out, prefix_len, scale):
    """Checks the (shape, stride, dtype) of a call and packs the desc's head; bytes of workspace."""
    int32 = _torch().int32
    name = "sdpa_shared_prefix"
    if len(q[0]) != 3 or len(k[0]) != 4 or v[0] != k[0]:
        raise ValueError(f"{name}: expected q [B, Hq, D] and pages [P, Hkv, page, D]")
    b, hq, d = q[0]
    pages, hk, page, dk = k[0]
    if dk != d:
        raise ValueError(f"{name}: K/V head_dim does not match Q")
    if len(table[0]) != 2 or len(lens[0]) != 1 or lens[0][0] != table[0][0]:
        raise ValueError(f"{name}: expected table [n, width] and lens [n]")
    if slots is not None and slots[0] != (b,):
        raise ValueError(f"{name}: slots must name one row per sequence")
    if out is None:
        out = (q[0], (hq * d, d, 1), q[2])
    elif out[0] != q[0]:
        raise ValueError(f"{name}: out must have q's shape")
    dtype = _check_rows(name, q[2], q, k, v, out)
    if not _dense(k[0][1:], k[1][1:]) or not _dense(v[0][1:], v[1][1:]):
        raise ValueError(f"{name}: a page must be contiguous")
    k_page, v_page = (x[1][0] if pages > 1 else hk * page * d for x in (k, v))
    for shape, stride, other in (table, lens) + (() if slots is None else (slots,)):
        if other != int32 or not _dense(shape, stride):
            raise ValueError(f"{name}: tables, lengths and slots are contiguous int32 tensors")
    head = _SHARED_HEAD.pack(b, hq, hk, d, page, pages, table[0][1], table[0][0], prefix_len,
                             *q[1][:2], *out[1][:2], k_page, v_page,
                             1.0 / math.sqrt(d) if scale is None else scale, dtype)
    need = ctypes.c_size_t()
    _launch(index, "enigma_sdpa_shared_prefix_workspace_bytes", head + _SHARED_PTRS.pack(*([0] * 9)),
            ctypes.byref(need))
    return head, need.value


def sdpa_shared_prefix(q, k_pages, v_pages, table, lens, prefix_len: int = 0, slots=None,
                       scale: Optional[float] = None, out=None, workspace=None):
    """One new token per sequence over a paged cache whose sequences share their first tokens.

    q [B, Hq, D]; k_pages / v_pages [pages, Hkv, page, D] (one layer of a cache); table
    [n, width] int32 page numbers, lens [n] int32; sequence b uses row slots[b] (default: row
    b).  Sequence b attends to its first lens keys; those below prefix_len are the same for
    the whole batch and are read through sequence 0's row, for many sequences at once on the tensor
    cores (bf16, heads of 64 or 128, aligned rows).  A sequence without keys gives zeros.  Which kernels run
    depends on the table's width, the most keys that a row could hold: a table no wider than its
    sequences need is faster.  workspace: a uint8 tensor to use instead of an allocation per call (as
    many bytes as enigma_sdpa_shared_prefix_workspace_bytes says).  Returns out [B, Hq, D].
    """
    index = _same_device("sdpa_shared_prefix", q, k_pages, v_pages, table, lens)
    head, need = _shared_head(
        index, (q.shape, q.stride(), q.dtype), (k_pages.shape, k_pages.stride(), k_pages.dtype),
        (v_pages.shape, v_pages.stride(), v_pages.dtype),
        (table.shape, table.stride(), table.dtype), (lens.shape, lens.stride(), lens.dtype),
        None if slots is None else (slots.shape, slots.stride(), slots.dtype),
        None if out is None else (out.shape, out.stride(), out.dtype), prefix_len, scale)
    if out is None:
        out = _contiguous_like(q)
    else:
        _same_device("sdpa_shared_prefix", q, out)
    ws, ws_bytes, keep = _scratch("sdpa_shared_prefix", workspace, need, q)
    if slots is not None:
        _same_device("sdpa_shared_prefix", q, slots)
    desc = head + _SHARED_PTRS.pack(table.data_ptr(), lens.data_ptr(),
                                    0 if slots is None else slots.data_ptr(), q.data_ptr(),
                                    k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), ws,
                                    ws_bytes)
    _launch(index, "enigma_sdpa_shared_prefix", desc, _raw_stream(index))
    return out


# enigma_sdpa_quantized_desc: sizes and strides, scale and types; then pointers.
_CODES_HEAD = struct.Struct("16qf3i")
_CODES_PTRS = struct.Struct("11Q")


def _code_of(dtype) -> int:
    torch = _torch()
    if dtype == torch.int8:
        return _native.CODE_INT8
    if dtype == torch.float8_e4m3fn:
        return _native.CODE_E4M3
    raise TypeError(f"unsupported codes {dtype}: expected int8 or float8_e4m3fn")


@functools.lru_cache(maxsize=1024)
def _quantized_head(index, q, k, v, ks, vs, table, lens, slots, out, scale):
    """Checks the (shape, stride, dtype) of a call and packs the desc's head; bytes of workspace."""
    torch = _torch()
    name = "sdpa_quantized"
    if len(q[0]) != 3 or len(k[0]) != 4 or v[0] != k[0]:
        raise ValueError(f"{name}: expected q [B, Hq, D] and pages [P, Hkv, page, D]")
    b, hq, d = q[0]
    pages, hk, page, dk = k[0]
    if dk != d:
        raise ValueError(f"{name}: K/V head_dim does not match Q")
    if v[2] != k[2]:
        raise TypeError(f"{name}: K and V must share a dtype")
    code = _code_of(k[2])
    parts = page // _native.SCALE_BLOCK
    for x in (ks, vs):
        if x[0] != (pages, hk, parts) or x[2] != torch.float32:
            raise ValueError(f"{name}: scales are fp32 [P, Hkv, page / {_native.SCALE_BLOCK}]")
    if len(table[0]) != 2 or len(lens[0]) != 1 or lens[0][0] != table[0][0]:
        raise ValueError(f"{name}: expected table [n, width] and lens [n]")
    if b > table[0][0] if slots is None else slots[0] != (b,):
        raise ValueError(f"{name}: slots must name one row per sequence")
    if out is None:
        out = (q[0], (hq * d, d, 1), q[2])
    elif out[0] != q[0]:
        raise ValueError(f"{name}: out must have q's shape")
    dtype = _check_rows(name, q[2], q, out)
    _check_distinct(name, out)
    if not all(_dense(x[0][1:], x[1][1:]) for x in (k, v, ks, vs)):
        raise ValueError(f"{name}: a page and its scales must be contiguous")
    strides = [x[1][0] if pages > 1 else math.prod(x[0]) for x in (k, v, ks, vs)]
    for shape, stride, other in (table, lens) + (() if slots is None else (slots,)):
        if other != torch.int32 or not _dense(shape, stride):
            raise ValueError(f"{name}: tables, lengths and slots are contiguous int32 tensors")
    head = _CODES_HEAD.pack(b, hq, hk, d, page, pages, table[0][1], table[0][0], *q[1][:2],
                            *out[1][:2], *strides, 1.0 / math.sqrt(d) if scale is None else scale,
                            dtype, code, 0)
    need = ctypes.c_size_t()
    _launch(index, "enigma_sdpa_quantized_workspace_bytes", head + _CODES_PTRS.pack(*([0] * 11)),
            ctypes.byref(need))
    return head, need.value


def sdpa_quantized(q, k_pages, v_pages, k_scale, v_scale, table, lens, slots=None,
                   scale: Optional[float] = None, out=None, workspace=None):
    """One new token per sequence over a paged cache held in 8-bit codes.

    q [B, Hq, D], bf16 or fp32; k_pages / v_pages [pages, Hkv, page, D], int8 or float8_e4m3fn (one
    layer of a kv_cache.QuantizedKVCache); k_scale / v_scale [pages, Hkv, page / 16] fp32: code x of
    a block of 16 tokens stands for x * scale (finite; a weight times its scale is held to 2^-34 of the
    largest |v_scale| beside it in bf16, 2^-40 in fp32).  table [n, width] int32 page numbers, lens [n] int32;
    sequence b uses row slots[b] (default: row b) and attends to its first lens keys, all read as
    its own (sequences that share pages find them in L2).  A sequence without keys gives zeros, a
    key without a page is zeros.  D is a multiple of 16 up to 256, page 16, 32, 64 or 128.
    workspace: a uint8 tensor to use instead of an allocation per call (as many bytes as
    enigma_sdpa_quantized_workspace_bytes says).  Returns out [B, Hq, D] of q's type.
    """
    name = "sdpa_quantized"
    index = _same_device(name, q, k_pages, v_pages, k_scale, v_scale, table, lens)
    head, need = _quantized_head(
        index, (q.shape, q.stride(), q.dtype), (k_pages.shape, k_pages.stride(), k_pages.dtype),
        (v_pages.shape, v_pages.stride(), v_pages.dtype),
        (k_scale.shape, k_scale.stride(), k_scale.dtype),
        (v_scale.shape, v_scale.stride(), v_scale.dtype),
        (table.shape, table.stride(), table.dtype), (lens.shape, lens.stride(), lens.dtype),
        None if slots is None else (slots.shape, slots.stride(), slots.dtype),
        None if out is None else (out.shape, out.stride(), out.dtype), scale)
    return _sdpa_quantized(index, head, need, [x.data_ptr() for x in (
        k_pages, v_pages, k_scale, v_scale, table, lens)], q, slots, out, workspace)


def _sdpa_quantized(index, head, need, pages, q, slots, out, workspace):
    """The launch, of checked sizes and types: `pages` holds the addresses of K's and V's pages, their
    scales, the table and the lengths, on device `index`."""
    name = "sdpa_quantized"
    if out is None:
        out = _contiguous_like(q)
    for t in (q, out, slots):
        if t is not None and t.get_device() != index:
            raise ValueError(f"{name}: all tensors must be on the same device")
    ws, ws_bytes, keep = _scratch(name, workspace, need, q)
    k, v, ks, vs, table, lens = pages
    desc = head + _CODES_PTRS.pack(table, lens, 0 if slots is None else slots.data_ptr(), q.data_ptr(),
                                   k, v, ks, vs, out.data_ptr(), ws, ws_bytes)
    _launch(index, "enigma_sdpa_quantized", desc, _raw_stream(index))
    return out


def rope_frequencies(rotary_dim: int, theta: float = 1e6, scaling: Optional[dict] = None):
    """(radians per position of each pair, factor on cos and sin), in Python's 64-bit floats.

    Pair i of n / 2 turns by w_i = theta^(-2 i / n).  scaling stretches contexts:
      {"type": "linear", "factor": f}: w_i / f;
      {"type": "ntk", "factor": f}: theta f^(n / (n - 2)) in place of theta;
      {"type": "yarn", "factor": f, "original_len": L, "beta_fast": 32, "beta_slow": 1}: pairs that
        turn more than beta_fast times over L positions keep w_i, those below beta_slow get w_i / f,
        linearly in i between the two (at i(beta) = n ln(L / 2 pi beta) / 2 ln theta, rounded
        outwards); the factor is "attention_factor", by default 0.1 ln f + 1, or 1 for f up to 1;
      {"type": "bands", "factor": f, "original_len": L, "low": a, "high": b}: pairs that turn
        more than b times over L keep w_i, those below a get w_i / f, linearly in the number of
        turns between.
    """
    n = rotary_dim
    if n < 0 or n % 2:
        raise ValueError("rope: rotary_dim must be even")
    if not theta > 1.0 or not math.isfinite(theta):
        raise ValueError("rope: theta must be greater than 1")
    spec = dict(scaling or {"type": "none"})
    kind, f = spec.pop("type", None), float(spec.pop("factor", 1.0))
    if not f > 0.0 or not math.isfinite(f):
        raise ValueError("rope: the scaling's factor must be positive")
    if kind == "none" and f != 1.0:
        raise ValueError("rope: a factor without a scaling to use it")

    def take(*names, **defaults):
        values = [spec.pop(x) for x in names if x in spec]
        if len(values) != len(names):
            raise ValueError(f"rope: {kind} scaling needs {', '.join(names)}")
        values += [spec.pop(x, default) for x, default in defaults.items()]
        if spec:
            raise ValueError(f"rope: {kind} scaling does not take {', '.join(spec)}")
        return [None if x is None else float(x) for x in values]

    if kind == "ntk":
        take()
        if n > 2:
            theta = theta * f ** (n / (n - 2))
    w = [theta ** (-2.0 * i / n) for i in range(n // 2)]
    if kind in ("none", "ntk"):
        take()
        return w, 1.0
    if kind == "linear":
        take()
        return [x / f for x in w], 1.0
    if kind == "yarn":
        length, fast, slow, factor = take("original_len", beta_fast=32.0, beta_slow=1.0,
                                          attention_factor=None)
        if not (length > 0 and fast > 0 and slow > 0):
            raise ValueError("rope: yarn scaling's numbers must be positive")
        if fast < slow:
            raise ValueError("rope: yarn scaling needs beta_fast of at least beta_slow")
        at = [n * math.log(length / (beta * 2 * math.pi)) / (2 * math.log(theta))
              for beta in (fast, slow)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), n - 1)
        ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3))) for i in range(n // 2)]
        return ([x * (1 - r) + x / f * r for x, r in zip(w, ramp)],
                0.1 * math.log(max(f, 1.0)) + 1 if factor is None else factor)
    if kind == "bands":
        length, low, high = take("original_len", "low", "high")
        if not (length > 0 and high > low):
            raise ValueError("rope: bands scaling needs original_len > 0 and high > low")
        keep = [min(1.0, max(0.0, (length * x / (2 * math.pi) - low) / (high - low))) for x in w]
        return [x * r + x / f * (1 - r) for x, r in zip(w, keep)], 1.0
    raise ValueError(f"rope: no scaling is called {kind!r}")


class RopeTable:
    """What `rope` needs to know of a model: made once, used by every layer and call.

    head_dim; rotary_dim: how many of a head's first elements turn (default: all); layout "half"
    (element i pairs with i + rotary_dim / 2, as in the decode layer) or "interleaved" (2 i with
    2 i + 1); theta and scaling as in `rope_frequencies`, or frequencies: radians per position of
    each pair (then `factor` may be given too).
    """

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, theta: float = 1e6,
                 layout: str = "half", scaling: Optional[dict] = None, frequencies=None,
                 factor: float = 1.0, device="cuda"):
        torch = _torch()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if layout not in ("half", "interleaved"):
            raise ValueError("rope: layout is 'half' or 'interleaved'")
        if not 0 < head_dim <= 4096 or not 0 <= rotary_dim <= head_dim or rotary_dim % 2:
            raise ValueError("rope: rotary_dim must be even and at most head_dim, head_dim at most "
                             "4096")
        if frequencies is None:
            frequencies, more = rope_frequencies(rotary_dim, theta, scaling)
            factor = factor * more
        elif scaling is not None:
            raise ValueError("rope: scaling or frequencies, not both")
        frequencies = [float(x) for x in frequencies]
        if len(frequencies) != rotary_dim // 2:
            raise ValueError("rope: one frequency for each pair")
        if not all(map(math.isfinite, frequencies)) or not math.isfinite(factor):
            raise ValueError("rope: frequencies and factor must be finite")
        # Full turns per position, as 64-bit binary fractions (angles are modulo a full turn).
        turns = [round(math.fmod(x / (2 * math.pi), 1.0) * 2.0 ** 64) % (1 << 64)
                 for x in frequencies]
        self.head_dim, self.rotary_dim = int(head_dim), int(rotary_dim)
        self.layout, self.factor = layout, float(factor)
        self.frequencies = frequencies
        self.turns = torch.tensor([x - (1 << 64) if x >> 63 else x for x in turns],
                                  dtype=torch.int64).to(device)
        self.heads = {}          # checked calls' sizes, strides and types


# enigma_rope_desc: sizes and strides, factor and types; then pointers.
_ROPE_HEAD = struct.Struct("13qf5i")
_ROPE_PTRS = struct.Struct("6Q")


def _check_distinct(name, *tensors):
    """Outputs whose elements are all places of their own: no axis repeats or overlaps another."""
    for shape, stride, _ in tensors:
        reach = 1
        for s, n in sorted((s, n) for s, n in zip(stride, shape) if n > 1):
            if s < reach and 0 not in shape:
                raise ValueError(f"{name}: an output's elements overlap")
            reach = s * (n - 1) + reach


def _rope_head(table, q, k, positions, out_q, out_k, inverse):
    """Checks the (shape, stride, dtype) of a call with this table and packs the desc's head."""
    torch = _torch()
    shapes = "rope: expected q and k [tokens, heads, head_dim]"
    if len(q[0]) != 3:
        raise ValueError(shapes)
    if k is None:
        if out_k is not None:
            raise ValueError("rope: out_k without k")
        k, out_k = ((q[0][0], 0, q[0][-1]), (0, 0, 1), q[2]), None
    if len(k[0]) != 3 or q[0][0] != k[0][0] or q[0][2] != k[0][2]:
        raise ValueError(shapes)
    tokens, hq, d = q[0]
    if d != table.head_dim:
        raise ValueError(f"rope: the table was made for heads of {table.head_dim}")
    if positions[0] != (tokens,) or not _dense(positions[0], positions[1]):
        raise ValueError("rope: positions must hold one number per token")
    if positions[2] not in (torch.int32, torch.int64):
        raise TypeError("rope: positions are int32 or int64")
    outs = []
    for x, out in ((q, out_q), (k, out_k)):
        if out is None:
            out = (x[0], (x[0][1] * d, d, 1), x[2])
        elif out[0] != x[0]:
            raise ValueError("rope: an output must have its input's shape")
        outs.append(out)
    dtype = _check_rows("rope", q[2], q, k, *outs)
    _check_distinct("rope", *outs)
    return _ROPE_HEAD.pack(tokens, hq, k[0][1], d, table.rotary_dim, *q[1][:2], *k[1][:2],
                           *outs[0][1][:2], *outs[1][1][:2], table.factor, dtype,
                           _native.ROPE_HALF if table.layout == "half"
                           else _native.ROPE_INTERLEAVED, bool(inverse),
                           8 if positions[2] == torch.int64 else 4, 0)


def rope(q, k, positions, table: RopeTable, inverse: bool = False, out_q=None, out_k=None):
    """Queries and keys turned to their positions, in one launch.

    q [tokens, Hq, D], k [tokens, Hkv, D] or None, any token and head strides, e.g. slices of one
    fused projection's output; positions [tokens], int32 or int64 on the device (negative ones turn
    back).  inverse=True turns by the negative angle: the transpose, so it also takes a result's
    gradient to its input's.  out_q / out_k: tensors to write, which may be q and k themselves but not
    overlap them otherwise.  An angle is off by at most 2^-52 of position * frequency, less than its
    rounding to fp32 up to positions of about 2^29.  Returns (q, k) turned, or q alone without k.
    """
    key = ((q.shape, q.stride(), q.dtype), None if k is None else (k.shape, k.stride(), k.dtype),
           (positions.shape, positions.stride(), positions.dtype),
           None if out_q is None else (out_q.shape, out_q.stride(), out_q.dtype),
           None if out_k is None else (out_k.shape, out_k.stride(), out_k.dtype), inverse)
    head = table.heads.get(key)
    if head is None:
        head = _rope_head(table, *key)
        if len(table.heads) >= 64:
            table.heads.clear()
        table.heads[key] = head
    index = q.get_device()
    if (positions.get_device() != index or table.turns.get_device() != index or index not in _initialised
            or k is not None and k.get_device() != index
            or out_q is not None and out_q.get_device() != index
            or out_k is not None and out_k.get_device() != index):
        _same_device("rope", q, *(x for x in (positions, table.turns, k, out_q, out_k) if x is not None))
    if out_q is None:
        out_q = _contiguous_like(q)
    if k is not None and out_k is None:
        out_k = _contiguous_like(k)
    desc = head + _ROPE_PTRS.pack(positions.data_ptr(), table.turns.data_ptr(), q.data_ptr(),
                                  0 if k is None else k.data_ptr(), out_q.data_ptr(),
                                  0 if k is None else out_k.data_ptr())
    _launch(index, "enigma_rope", desc, _raw_stream(index))
    return out_q if k is None else (out_q, out_k)


def synchronize(device_index: int = 0) -> None:
    """Synchronize the device and raise if a kernel reported a device-side timeout."""
    ensure_device(device_index)
    _launch(device_index, "enigma_synchronize", None)
