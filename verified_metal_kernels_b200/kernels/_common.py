"""Argument checks shared by the kernel modules."""
import ctypes
import importlib.util
import os

import torch

from .. import _lib, build

_ENTRIES = ("vmk_prompt_workspace_bytes", "vmk_prompt", "vmk_prompt_paged", "vmk_accept", "vmk_pages_workspace_bytes",
            "vmk_pages_reserve", "vmk_pages_append_granted", "vmk_pages_fork", "vmk_pages_compact_granted", "vmk_pages_free", "vmk_pages_copy")
_calls = None


def need(t, name, dtype, shape=None, dims=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor (the kernels have no CPU path)")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected dtype {dtype}, got {t.dtype}")
    if dims is not None and t.dim() != dims:
        raise ValueError(f"{name}: expected {dims} dimensions, got shape {tuple(t.shape)}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: expected a C-contiguous tensor")
    return t


def stage_in(tensors):
    """Host tensors (pinned or not) -> device copies on the current stream; device tensors pass through.
    Returns (device tensors, any_host)."""
    out, any_host = [], False
    for t in tensors:
        if t is not None and not t.is_cuda:
            any_host = True
            t = t.to("cuda", non_blocking=True)
        out.append(t)
    return out, any_host


def need_on(t, name, dtype, shape, dev):
    """need(t, name, dtype, shape) on device `dev`, in one look where all is well."""
    if (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == dev and t.is_cuda and t.is_contiguous()):
        return t
    need(t, name, dtype, shape=shape)
    raise ValueError(f"{name}: expected a tensor on {dev}, got {t.device}")


def elsewhere(dev):
    """Whether `dev` is not the current device: the caller then makes it so and calls itself again (a `with` that does
    nothing costs as much as a check)."""
    return torch._C._cuda_getDevice() != dev.index


def calls():
    """The compiled form of the modules' ordinary calls (csrc/torch_calls.cpp), loaded on first use.  Its functions return
    None, having done nothing, for every call that is not ordinary.  It reads torch's tensors by the layout of the torch that
    built it and calls the C entry points by their place in _ENTRIES: one that was built from anything else is not loaded."""
    global _calls
    if _calls is None:
        path = os.path.join(_lib.HERE, "_vmk_torch.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: build it with `python -m verified_metal_kernels_b200.build`")
        if not build.calls_fresh():
            raise RuntimeError(f"{path} was built for another torch, Python or source: build it with "
                               "`python -m verified_metal_kernels_b200.build`")
        lib = _lib.lib()
        spec = importlib.util.spec_from_file_location("_vmk_torch", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.init(*[ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _ENTRIES])
        _calls = module
    return _calls


def handles(dev):
    """Torch's current stream on `dev` as an integer (no Stream object is built) and the address of the device's status word."""
    status = _lib.status_word(dev).data_ptr()
    calls().set_status(dev.index, status)
    return torch._C._cuda_getCurrentRawStream(dev.index), status


def scratch(nbytes, dev, stream):
    """Scratch of a call made while `dev` is the current device: address and size.  Its tensor may be let go at once: under
    capture the graph's memory pool gives it to later calls of the same stream only."""
    t = _lib.workspace(nbytes, dev, stream)
    return t.data_ptr(), t.numel()
