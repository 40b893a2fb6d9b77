"""CUDA-graph capture of a whole callable (the trunk), replayed with fresh inputs.

FoldForge's execution policy captures the trunk once and replays it
(``execution.cuda_graph`` with scope ``trunk``, ``src/foldforge/models/execution.py:196-260``).
The b200 kernels are capturable: they allocate nothing, never synchronise the host, and
take every buffer as an argument. Weights are packed on the eager warm-up call, before
capture.

A graph knows a packed weight image by its address alone, and a module replaces its image when its
weights change: what an op hands out under capture is kept here, by the :class:`GraphedCall` that
captures it or else (a capture of the caller's own) as long as the module lives. A replay goes on
reading the image it was captured with.
"""

from __future__ import annotations

import threading
from collections.abc import Callable, Iterator, Sequence
from contextlib import contextmanager
from weakref import WeakKeyDictionary

import torch
from torch import nn

Tensor = torch.Tensor
_holder = threading.local()  # .images: the list of the capture that runs on this thread
_of_modules: WeakKeyDictionary[nn.Module, list[Tensor]] = WeakKeyDictionary()


def capturing() -> bool:
    """Whether the current stream is being captured into a graph."""
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


@contextmanager
def holding(images: list[Tensor]) -> Iterator[None]:
    """Images that ops of this thread hand out under capture meanwhile go to ``images``."""
    before = getattr(_holder, "images", None)
    _holder.images = images
    try:
        yield
    finally:
        _holder.images = before


def keep_image(module: nn.Module, image: Tensor) -> None:
    """Keep an image of ``module`` that a graph being captured reads."""
    images = getattr(_holder, "images", None)
    if images is None:
        images = _of_modules.setdefault(module, [])
    if not any(kept is image for kept in images):
        images.append(image)


class GraphedCall:
    """``fn(*inputs)`` captured on static copies of ``example_inputs``.

    Calling the object copies the new inputs into the static buffers (same shapes and
    dtypes), replays the graph on the current stream and returns the static outputs
    (overwritten by the next call).
    """

    def __init__(self, fn: Callable[..., object], example_inputs: Sequence[Tensor], warmup: int = 1) -> None:
        self.fn = fn
        self.static_inputs = [t.clone() for t in example_inputs]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream), torch.no_grad():
            for _ in range(warmup):
                fn(*self.static_inputs)
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        self.images: list[Tensor] = []
        with torch.cuda.graph(self.graph), torch.no_grad(), holding(self.images):
            self.static_outputs = fn(*self.static_inputs)
        torch.cuda.synchronize()

    def replay(self) -> object:
        """Replay on the inputs already in :attr:`static_inputs`."""
        self.graph.replay()
        return self.static_outputs

    def __call__(self, *inputs: Tensor) -> object:
        for dst, src in zip(self.static_inputs, inputs, strict=True):
            dst.copy_(src, non_blocking=True)
        return self.replay()
