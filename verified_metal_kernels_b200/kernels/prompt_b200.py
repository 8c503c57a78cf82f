"""Kernel module for prompt attention on B200: whole prompts, or chunks of prompts over a cache.

Not one of the reference's three ops, which all decode (reference ops/spec.py:14-25 has the causal chain over a
cache's last positions, at most 32 of them): it is what fills the caches that they read.  Packed sequences of
different lengths, causal, grouped heads; contiguous keys or the paged cache of decode_b200.kernel_paged."""
import struct

import torch

from .. import _lib
from ._common import calls, elsewhere, handles, need, need_on, scratch, stage_in


def _rows(t, name, dtype):
    """A (tokens, heads, 128) tensor whose innermost axis is contiguous; the other two may have any stride that is a
    positive multiple of 8 elements (a view of a fused q/k/v projection, for instance)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch tensor, got {type(t).__name__}")
    if t.dtype is dtype and t.dim() == 3 and t.is_cuda and t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor (the kernels have no CPU path)")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected dtype {dtype}, got {t.dtype}")
    if t.dim() != 3:
        raise ValueError(f"{name}: expected 3 dimensions, got shape {tuple(t.shape)}")
    if t.numel():
        if t.stride(2) != 1 and t.shape[2] > 1:
            raise ValueError(f"{name}: expected a contiguous innermost axis")
        for axis in (0, 1):
            if t.shape[axis] > 1 and (t.stride(axis) <= 0 or t.stride(axis) % 8 != 0):
                raise ValueError(f"{name}: the stride of axis {axis} must be a positive multiple of 8 elements")
        if t.data_ptr() % 16:
            raise ValueError(f"{name}: expected a 16-byte aligned tensor")
    return t


def _strides(*tensors):
    """Token and head strides for the C call: null where every tensor is contiguous, else six (two) int64."""
    if all(t.is_contiguous() for t in tensors):
        return None
    return struct.pack(f"{2 * len(tensors)}q", *[n for t in tensors for n in t.stride()[:2]])


def _common(q, cu_q):
    if not isinstance(q, torch.Tensor) or q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("q: expected a float16 or bfloat16 tensor")
    _rows(q, "q", q.dtype)
    need(cu_q, "cu_q", torch.int32, dims=1)
    if cu_q.shape[0] < 1:
        raise ValueError("cu_q: expected at least one entry")
    return q.dtype, q.shape[0], q.shape[1], q.shape[2], cu_q.shape[0] - 1


def _same_device(dev, **tensors):
    for name, t in tensors.items():
        if t.device != dev:
            raise ValueError(f"{name}: expected a tensor on {dev}, got {t.device}")


def kernel(q, k, v, cu_q, cu_k=None, causal=True, check=False):
    """q (Tq,Hq,128), k/v (Tk,Hkv,128) fp16 or bf16, packed by cu_q and cu_k (S+1,) int32 (cu_k None: the same as
    cu_q) -> (Tq,Hq,128).  Query i of a sequence with nq queries and nk keys sees its keys j <= nk - nq + i, with
    causal=False all of them.  A query that sees no key gets zeros, and so do rows outside [cu_q[0], cu_q[-1]).
    q, k and v may be views (see the strides that _rows allows).  Host tensors are copied in and the result returned
    on the host (with the device status word checked; device-resident calls check it only with check=True)."""
    if not check:
        out = calls().prompt(q, k, v, cu_q, cu_k, causal)
        if out is not None:
            return out
    (q, k, v, cu_q, cu_k), host = stage_in([q, k, v, cu_q, cu_k])
    dt, Tq, Hq, D, S = _common(q, cu_q)
    _rows(k, "k", dt)
    Tk, Hkv = k.shape[0], k.shape[1]
    _rows(v, "v", dt)
    if tuple(k.shape) != (Tk, Hkv, D) or v.shape != k.shape:
        raise ValueError(f"k, v: expected shape (keys, kv heads, {D}), got {tuple(k.shape)} and {tuple(v.shape)}")
    dev = q.device
    cu_k = cu_q if cu_k is None else need_on(cu_k, "cu_k", torch.int32, (S + 1,), dev)
    if k.device != dev or v.device != dev or cu_q.device != dev:
        _same_device(dev, k=k, v=v, cu_q=cu_q)
    lib = _lib.lib()
    if elsewhere(dev):
        with torch.cuda.device(dev):
            return kernel(q, k, v, cu_q, cu_k, causal, check)
    stream, status = handles(dev)
    out = q.new_empty(q.shape)
    nbytes = lib.vmk_prompt_workspace_bytes(S, Tq, Tk, Hq, Hkv, D) if Hkv else 0
    if nbytes == 0:
        raise _lib.VmkError(-2, "prompt: unsupported shape")
    ws = scratch(nbytes, dev, stream)
    rc = lib.vmk_prompt(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), _strides(q, k, v),
                        out.data_ptr(), S, Tq, Tk, Hq, Hkv, D, 1 if causal else 0, 1 if dt == torch.bfloat16 else 0,
                        *ws, status, stream)
    _lib.check(rc, "vmk_prompt")
    return _lib.finish(out, host, check, dev, "vmk_prompt")


def kernel_paged(q, k_pages, v_pages, page_table, cu_q, lens, causal=True, check=False):
    """The same over a paged cache: k_pages / v_pages (pages,Hkv,page_size,128), page_table (S,T) int32, lens (S,)
    int32 the keys of each sequence, its new tokens (already appended) included; page_size a multiple of 64."""
    if not check:
        out = calls().prompt_paged(q, k_pages, v_pages, page_table, cu_q, lens, causal)
        if out is not None:
            return out
    dt, Tq, Hq, D, S = _common(q, cu_q)
    need(k_pages, "k_pages", dt, dims=4)
    pages, Hkv, page_size = k_pages.shape[0], k_pages.shape[1], k_pages.shape[2]
    need(k_pages, "k_pages", dt, shape=(pages, Hkv, page_size, D))
    need(v_pages, "v_pages", dt, shape=(pages, Hkv, page_size, D))
    need(page_table, "page_table", torch.int32, dims=2)
    T = page_table.shape[1]
    dev = q.device
    need_on(page_table, "page_table", torch.int32, (S, T), dev)
    need_on(lens, "lens", torch.int32, (S,), dev)
    if page_size == 0 or page_size % 64 != 0:
        raise ValueError("page_size must be a multiple of 64")
    if k_pages.device != dev or v_pages.device != dev or cu_q.device != dev:
        _same_device(dev, k_pages=k_pages, v_pages=v_pages, cu_q=cu_q)
    lib = _lib.lib()
    if elsewhere(dev):
        with torch.cuda.device(dev):
            return kernel_paged(q, k_pages, v_pages, page_table, cu_q, lens, causal, check)
    stream, status = handles(dev)
    out = q.new_empty(q.shape)
    nbytes = lib.vmk_prompt_workspace_bytes(S, Tq, T * page_size, Hq, Hkv, D) if Hkv else 0
    if nbytes == 0:
        raise _lib.VmkError(-2, "prompt: unsupported shape")
    ws = scratch(nbytes, dev, stream)
    rc = lib.vmk_prompt_paged(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), pages, page_size,
                              T, cu_q.data_ptr(), lens.data_ptr(), _strides(q), out.data_ptr(), S, Tq, Hq, Hkv, D,
                              1 if causal else 0, 1 if dt == torch.bfloat16 else 0, *ws,
                              status, stream)
    _lib.check(rc, "vmk_prompt_paged")
    return _lib.finish(out, False, check, dev, "vmk_prompt_paged")
