"""The short ways from a public function to its C entry.

A ``torch.library.custom_op`` costs 15-25 us of host time per call (dispatcher,
autograd and in-place bookkeeping), several times the kernels of a decode step.
So in plain eager mode, with nothing to differentiate, the public functions of
the verification operators take one of two shorter ways:

* the ``_fast`` module (csrc/fast_call.cpp) checks, allocates and launches
  without Python; it returns None when anything is not plain or not as the
  operator wants it (or the module was not built);
* then the Python implementation runs directly (it raises for what is wrong).

Under torch.compile, torch.jit.trace, fake tensors, dispatch modes, functorch
transforms, forward derivatives and for inputs that require a gradient they go
through the registered operator, whose kernel is the same Python implementation (rotary has its gradient
in the shorter ways too).
"""

from __future__ import annotations

import ctypes
import importlib.util
import warnings
from pathlib import Path
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib

_PLAIN = (torch.Tensor, torch.nn.Parameter)
_modes = torch._C._len_torch_dispatch_stack
_interpreter = torch._C._functorch.peek_interpreter_stack
_tracing = torch._C._get_tracing_state
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_device = getattr(torch._C, "_cuda_getDevice", None)
compiling = torch.compiler.is_compiling

# the order of Entries in csrc/fast_call.cpp
_ENTRIES = ("b200kv_rotary", "b200kv_kv_store", "b200kv_kv_load", "b200kv_tree_mask", "b200kv_tree_workspace_bytes",
            "b200kv_tree_attention", "b200kv_tree_commit")


class _Absent:
    """Stands in for the module where it was not built: every call takes the Python way."""

    def __getattr__(self, name):
        return lambda *args: None


class _Unbound:
    """Stands in until the first call: loads the library and binds the module to it."""

    def __getattr__(self, name):
        global fast
        from .build import fast_name  # (here, so that `python -m torch_spyre_b200.build` is its only import)

        path = Path(__file__).resolve().parent / "lib" / fast_name()
        handle = _lib.lib()
        if path.exists():
            spec = importlib.util.spec_from_file_location("_fast", path)
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
            module.bind(*(ctypes.cast(getattr(handle, e), ctypes.c_void_p).value for e in _ENTRIES))
        else:
            warnings.warn(f"{path} is missing, calls go through Python (three times the host time): build it with "
                          "`python -m torch_spyre_b200.build`", RuntimeWarning, stacklevel=3)
            module = _Absent()
        fast = module
        return getattr(module, name)


fast = _Unbound()


def plain(t: torch.Tensor) -> bool:
    return type(t) in _PLAIN and t.is_cuda


def direct(*tensors) -> bool:
    """Whether a call on these tensors (None among them) may skip the dispatcher."""
    if compiling() or _modes() or _interpreter() is not None or forward_ad._current_level >= 0 or _tracing() is not None:
        return False
    grad = torch.is_grad_enabled()
    return all(t is None or (plain(t) and not (grad and t.requires_grad)) for t in tensors)


def flag_ptr(flag: Optional[torch.Tensor], device: torch.device) -> Optional[int]:
    """Address of an error flag, which a kernel on ``device`` may write to."""
    if flag is None:
        return None
    if flag.dtype != torch.int32 or flag.device != device or flag.numel() < 1:
        raise ValueError(f"error_flag must be an int32 tensor on {device}, got {flag.numel()} elements of {flag.dtype} "
                         f"on {flag.device}")
    return flag.data_ptr()


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
    torch.autograd.graph.increment_version([t for t in tensors if t is not None and not t.is_inference()])
