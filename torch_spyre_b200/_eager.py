"""The short way from a public function to its C entry.

A ``torch.library.custom_op`` costs 15-25 us of host time per call (dispatcher,
autograd and in-place bookkeeping), several times the kernels of a decode step.
In plain eager mode the public functions therefore call their implementation
directly; under torch.compile, fake tensors, dispatch modes or functorch
transforms they go through the registered operator, whose kernel is the same
implementation.
"""

from __future__ import annotations

import torch

from . import _lib

_PLAIN = (torch.Tensor, torch.nn.Parameter)
_modes = torch._C._len_torch_dispatch_stack
_interpreter = torch._C._functorch.peek_interpreter_stack
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_device = getattr(torch._C, "_cuda_getDevice", None)


def direct(x: torch.Tensor) -> bool:
    """Whether a call on x may skip the dispatcher."""
    return (type(x) in _PLAIN and x.is_cuda and not _modes() and _interpreter() is None
            and not torch.compiler.is_compiling())


def launch(name: str, device: torch.device, *args) -> None:
    """Calls entry ``name`` with args and the device's current stream, on that device."""
    index = device.index
    if index == _device():
        status = getattr(_lib.lib(), name)(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            status = getattr(_lib.lib(), name)(*args, _stream(index))
    if status:
        _lib.check(status, name)


def written(*tensors) -> None:
    """Marks tensors as changed in place, as the registered operator does."""
    torch.autograd.graph.increment_version([t for t in tensors if t is not None])
