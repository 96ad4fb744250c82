"""Streams that nothing else in the process is given."""

from __future__ import annotations

import atexit

import torch

from ..ops import get_extension


def own_stream(device) -> torch.cuda.Stream:
    """A stream outside torch's pool, at the default priority, kept until the
    process ends.

    The math libraries keep one workspace a stream, and graphs hold it by
    address: two that replay side by side must not be captured on one stream.
    torch.cuda.Stream() deals out 32 of them in turn, so the 33rd is the first
    again, and torch's own capture stream is one of them."""
    ext = get_extension()
    with torch.cuda.device(device):
        ptr = ext.create_stream()
    # a leaked queue ends a profiler's teardown with a segmentation fault
    atexit.register(ext.destroy_stream, ptr)
    return torch.cuda.ExternalStream(ptr, device=device)
