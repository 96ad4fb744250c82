"""Streams to capture graphs on that replay side by side."""

from __future__ import annotations

import gc
import weakref

import torch

POOL = 32  # streams that torch deals out in turn

# by owner, not by stream: torch's streams leave weak references dangling
_taken: "weakref.WeakKeyDictionary" = weakref.WeakKeyDictionary()


def _number(stream):
    return stream.device_index, stream.stream_id


def capture_stream(owner, device) -> torch.cuda.Stream:
    """A stream for `owner` to capture graphs on, as long as it lives: no other
    owner's, nor the one that torch captures on where it is not told which.

    The math libraries keep one workspace a stream and a graph holds it by
    address, so graphs captured on one stream must not replay side by side.
    torch.cuda.Stream() alone does not keep them apart: the 33rd is the first
    again.

    Streams are told apart by torch's number, not by their address, for which
    torch would make them here.  Which hardware queues the branches of replayed
    graphs fall on goes by the streams that were made before them: made before
    the actor's and learner's masked queues, or as two more outside the pool, the
    colocated round falls from 5.9 M frames a second to 4.6."""
    if torch.cuda.graph.default_capture_stream is None:
        # chosen at the first such capture otherwise, perhaps one that is taken
        torch.cuda.graph.default_capture_stream = torch.cuda.Stream(device)
    for _ in range(2):
        taken = {*_taken.values(), _number(torch.cuda.graph.default_capture_stream)}
        for _ in range(POOL):
            stream = torch.cuda.Stream(device)
            if _number(stream) not in taken:
                _taken[owner] = _number(stream)
                return stream
        gc.collect()  # owners that only refer to each other
    raise RuntimeError(f"{len(_taken)} owners of graphs hold all of torch's streams")
