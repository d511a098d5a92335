"""Calling the native library: the stream and device of a launch, and refusals."""

from __future__ import annotations

import torch

from cernels_amd._native import check


def stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: stream(torch.device("cuda", i)))


def launch(what: str, device_index: int, fn, *args) -> None:
    """One native call on the current stream of the tensors' device, which is made current where it is not."""
    if torch.cuda.current_device() == device_index:
        st = fn(*args, _raw_stream(device_index))
    else:
        with torch.cuda.device(device_index):
            st = fn(*args, _raw_stream(device_index))
    check(st, what)


def require(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)
