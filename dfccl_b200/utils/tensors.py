"""Views of symmetric-heap memory as torch tensors (no copy, no ownership)."""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Sequence

import numpy as np
import torch
import torch.autograd.forward_ad as forward_ad

from .. import native as nv

_TORCH_TO_NCCL = {
    torch.int8: nv.INT8, torch.uint8: nv.UINT8, torch.int32: nv.INT32, torch.int64: nv.INT64,
    torch.float16: nv.FLOAT16, torch.float32: nv.FLOAT32, torch.float64: nv.FLOAT64, torch.bfloat16: nv.BFLOAT16,
}


def nccl_dtype(dt: torch.dtype) -> int:
    try:
        return _TORCH_TO_NCCL[dt]
    except KeyError:
        raise TypeError(f"{dt} has no collective datatype") from None


def raw_stream(device: torch.device) -> int:
    """Handle of the device's current stream: what ``torch.cuda.current_stream(device).cuda_stream`` gives, without making
    a Stream object for every launch (2.2 us of host time)."""
    index = device.index
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if index is None else index)


def stream_of(t: torch.Tensor) -> int:
    """The same for the device that holds ``t``, a GPU."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


_HERE = contextlib.nullcontext()


def on_device(device: torch.device):
    """Makes ``device`` the current one for a launch on its stream, where it is not already (a launch on another device's
    stream is refused by the runtime)."""
    return _HERE if device.index is None or device.index == torch.cuda.current_device() else torch.cuda.device(device.index)


def refuse_tangents(*tensors) -> None:
    """Kernels that read by address would leave a forward-mode tangent behind without a word; tensors may be None."""
    if forward_ad._current_level < 0:                   # tangents live inside a level only (asked of each tensor, it is 1 us of a launch)
        return
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("no forward-mode derivative of this operator; its gradients come from a backward pass")


class _CudaBlob:
    """Minimal ``__cuda_array_interface__`` provider for a raw device range."""

    def __init__(self, ptr: int, nbytes: int):
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "data": (ptr, False), "version": 2}


def tensor_from_ptr(ptr: int, shape: Sequence[int], dtype: torch.dtype, device) -> torch.Tensor:
    """Tensor over ``prod(shape)`` elements of ``dtype`` starting at device (or host) address ``ptr``.
    The memory stays owned by the heap; the caller keeps it alive."""
    n = 1
    for s in shape:
        n *= int(s)
    nbytes = n * torch.empty((), dtype=dtype).element_size()
    device = torch.device(device)
    if device.type == "cuda":
        raw = torch.as_tensor(_CudaBlob(ptr, max(nbytes, 1)), device=device)
    else:
        buf = (C.c_uint8 * max(nbytes, 1)).from_address(ptr)
        raw = torch.from_numpy(np.frombuffer(buf, dtype=np.uint8))
    return raw[:nbytes].view(dtype).view(*shape)


class HeapTensorPool:
    """Allocates tensors from a communicator's symmetric heap and frees them together."""

    def __init__(self, comm: nv.Comm, device):
        self.comm, self.device, self._ptrs = comm, torch.device(device), []

    def empty(self, shape: Sequence[int], dtype: torch.dtype) -> torch.Tensor:
        n = 1
        for s in shape:
            n *= int(s)
        nbytes = max(1, n * torch.empty((), dtype=dtype).element_size())
        p = self.comm.alloc(nbytes)
        self._ptrs.append(p)
        return tensor_from_ptr(p, shape, dtype, self.device)

    def zeros(self, shape, dtype):
        return self.empty(shape, dtype).zero_()

    def release(self):
        for p in self._ptrs:
            self.comm.free(p)
        self._ptrs.clear()
