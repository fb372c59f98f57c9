"""Torch-side plumbing for the HIP ops: device checks, dtype codes, streams,
status words.  torch only provides device memory and the current stream."""
from __future__ import annotations

import torch

from . import _lib
from .errors import IntegrityError

DTYPE_CODE = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}


def dtype_code(dt):
    if dt not in DTYPE_CODE:
        raise IntegrityError(f"unsupported dtype {dt}")
    return DTYPE_CODE[dt]


def require_gpu(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise IntegrityError("NSN HIP ops require GPU tensors; there is no CPU fallback")


def require_current(*tensors):
    """Work goes to the current device's stream: its tensors must be there.
    Returns the device's index."""
    dev = torch.cuda.current_device() if tensors[0].is_cuda else -1
    for t in tensors:
        if t.get_device() != dev or dev < 0:
            require_gpu(t)
            raise IntegrityError(f"Tensor on {t.device}, but the current device is cuda:{dev}")
    return dev


def stream():
    """The current stream of the current device as a raw hipStream_t (an int).
    torch's raw accessor costs ~1 µs; ``torch.cuda.current_stream()`` builds a
    Stream object and resolves the device index (~11 µs per call)."""
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def capturing():
    """Work of the current stream is recorded into a HIP graph, not run."""
    return torch.cuda.is_current_stream_capturing()


def ptr(t):
    return None if t is None else t.data_ptr()


def new_status(device):
    return torch.zeros(1, dtype=torch.int32, device=device)


def require_status(status, dev):
    if status.dtype != torch.int32 or status.numel() < 1 or status.get_device() != dev:
        raise IntegrityError(f"Status word (int32 on cuda:{dev})")
    return status


def read_status(status):
    """Synchronising read of a device status word."""
    return int(status.item())


def norm_order(x):
    """Order of torch-CPU's vector_norm on ``x.float()`` (see include/nsn_hip.h).

    ``x.float()`` keeps ``x``'s strides when ``x`` is non-overlapping and
    dense (and is ``x`` itself for fp32); its last-dim stride decides between
    the 8-lane contiguous reduction and the sequential one.
    """
    if x.dtype == torch.float32:
        st = x.stride(-1)
    else:
        st = torch.empty_like(x, dtype=torch.float32, device="meta").stride(-1)
    return _lib.NORM_LANES8 if (st == 1 or x.shape[-1] == 1) else _lib.NORM_SEQUENTIAL
