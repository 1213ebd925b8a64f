"""Torch buffer plumbing for the C ABI: pointers, streams, checks."""

from __future__ import annotations

import torch

from . import _lib


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def stream_of(t: torch.Tensor) -> int:
    """The current torch stream handle on ``t``'s device (launches are stream-ordered)."""
    return torch.cuda.current_stream(t.device).cuda_stream


def require_cuda(*ts: torch.Tensor) -> torch.device:
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise _lib.DSparkUnsupported(
                _lib.ERR_UNSUPPORTED, f"tensor on {t.device}: dspark kernels run on CUDA only "
                "(there is no CPU path)")
        dev = t.device if dev is None else dev
        if t.device != dev:
            raise _lib.DSparkError(_lib.ERR_ARG, "tensors on different devices")
    assert dev is not None
    _lib.ensure_init(dev.index if dev.index is not None else torch.cuda.current_device())
    return dev


def elem_strides(t: torch.Tensor, n: int = 3) -> list[int]:
    return [int(s) for s in t.stride()[:n]]


def on_device(first: torch.Tensor, *rest: torch.Tensor | None) -> int:
    """The current stream on the CUDA device of ``first``, with every other tensor (``None`` skipped)
    on that device. Launches go to the current device, so it has to be that one."""
    dev = first.get_device()
    if dev < 0:
        raise _lib.DSparkUnsupported(
            _lib.ERR_UNSUPPORTED, f"tensor on {first.device}: dspark kernels run on CUDA only "
            "(there is no CPU path)")
    for t in rest:
        if t is not None and t.get_device() != dev:
            raise _lib.DSparkError(_lib.ERR_ARG, f"tensors on {first.device} and {t.device}")
    if dev != torch._C._cuda_getDevice():
        raise _lib.DSparkError(_lib.ERR_ARG, f"tensors on {first.device}, which is not the current device")
    if dev not in _lib._inited:
        _lib.ensure_init(dev)
    return torch._C._cuda_getCurrentRawStream(dev)


def int32(name: str, t: torch.Tensor | None, n: int | None = None) -> int:
    """The address of ``t``, checked to be contiguous int32 (and of ``n`` values): what the kernels
    index. 0 for ``None``."""
    if t is None:
        return 0
    if t.dtype is not torch.int32 or not t.is_contiguous():
        raise _lib.DSparkError(_lib.ERR_ARG, f"{name} must be contiguous int32, got {t.dtype}")
    if n is not None and t.numel() != n:
        raise _lib.DSparkError(_lib.ERR_ARG, f"{name} has {t.numel()} values, {n} are needed")
    return t.data_ptr()
