"""Host side of the serving operators, whose kernels often take less time than a call of them: entry points that take their
arguments' fields packed at once; and what asks, for them and in ``kernels``, whether a call needs torch's dispatcher."""
from __future__ import annotations

import ctypes
import struct

import torch
from torch import Tensor

from . import _lib

_compiling = torch.compiler.is_compiling
_dispatch_modes, _tracing = torch._C._len_torch_dispatch_stack, torch._C._get_tracing_state
_transform, _grad_mode = torch._C._functorch.peek_interpreter_stack, torch.is_grad_enabled
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_Parameter = torch.nn.Parameter


def watched() -> bool:
    """Whether torch has to see every operator: tracing (torch.compile, torch.jit.trace), a dispatch mode, a functorch transform."""
    return _compiling() or _dispatch_modes() > 0 or _tracing() is not None or _transform() is not None


def plain(first: Tensor, *others) -> bool:
    """Whether a call with these tensors (or Nones) needs nothing of the dispatcher (``kernels.dispatcher_needed`` is the same of any
    arguments), and all are on one GPU: the operator's body then need not look at that again."""
    if watched():
        return False
    if type(first) is not Tensor or not first.is_cuda:
        return False
    dev, grad = first.get_device(), _grad_mode()
    if grad and first.requires_grad:
        return False
    for t in others:
        if t is not None and (t.get_device() != dev or (type(t) is not Tensor and type(t) is not _Parameter) or (grad and t.requires_grad)):
            return False
    return True


class Entry:
    """The C entry point ``name``, called with the fields of its argument struct (``fields``: their ``struct`` format, as the
    ctypes declaration ``declared`` in ``_lib`` lays them out) on a device's current stream."""

    __slots__ = ("name", "pack", "size", "declared", "stream", "fn")

    def __init__(self, name: str, fields: str, declared: str, stream: bool = True):
        form = struct.Struct("@" + fields)
        self.name, self.pack, self.size, self.declared, self.stream, self.fn = name, form.pack, form.size, declared, stream, None

    def _bind(self):
        _lib.entry(self.name)  # raises if the library is missing or lacks it
        if self.size != ctypes.sizeof(getattr(_lib, self.declared)):
            raise RuntimeError(f"{self.name}: packed arguments of {self.size} bytes do not match {self.declared}")
        fn = _lib.load()[self.name]  # a handle of its own, with its own argument types
        fn.restype = _lib.SIGNATURES[self.name][0]
        fn.argtypes = [ctypes.c_char_p, ctypes.c_void_p] if self.stream else [ctypes.c_char_p]
        self.fn = fn  # last: another thread calls whatever it finds here

    def __call__(self, op: str, dev: int, *values):
        if self.fn is None:
            self._bind()
        args = self.pack(*values)
        if not self.stream:
            return self.fn(args)
        if dev == _current_device():
            rc = self.fn(args, _raw_stream(dev))
        else:
            with torch.cuda.device(dev):
                rc = self.fn(args, _raw_stream(dev))
        if rc:
            _lib.check(rc, op)
