"""Python face of the C ABI, in the calling style of the reference's own ctypes
harness (tests/conftest.py:141-173, ``ProcWrapper``): positional arguments,
``None`` for the context, ints for sizes, arrays for tensors -- e.g.
``lib.sgemm_exo(None, M, N, K, A, B, C)`` exactly as one would call the library
``exocc`` generates.  Tensors may be numpy arrays (host memory: staged to the
GPU and back inside the call) or torch CUDA tensors (used in place, on torch's
current stream).  Results are written into the output argument.

Errors: the C functions return void (as the reference's do); this wrapper reads
the library's error side channel after each call and raises ``ExoB200Error``.
"""
from __future__ import annotations

import ctypes
import operator
import threading

import numpy as np

from . import _lib

try:  # the fast path of CheckedProc (csrc/call.cpp), where it has been built
    from . import _call
except ImportError:
    _call = None


class ExoB200Error(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"[{code}] {msg}")
        self.code = code


OK, ERR_INVALID_ARGUMENT, ERR_CUDA, ERR_TIMEOUT, ERR_UNSUPPORTED = range(5)
SGEMM_FFMA, SGEMM_3XTF32 = 0, 1


def _is_torch(x) -> bool:
    return type(x).__module__.startswith("torch") and hasattr(x, "data_ptr")


def _convert(arg, argtype, keepalive):
    """One argument, the way ProcWrapper._convert does it, plus torch tensors,
    Python floats for by-pointer scalars, and Context objects.  Temporaries that
    the C call reads through a pointer are appended to ``keepalive``, which the
    caller owns until the C function has returned."""
    if arg is None:
        return None
    if isinstance(arg, Context):
        return arg.handle
    if isinstance(arg, np.ndarray):
        if not arg.flags["C_CONTIGUOUS"]:
            raise ValueError("arrays must be C-contiguous (dense row-major)")
        return ctypes.c_void_p(arg.ctypes.data)
    if _is_torch(arg):
        if not arg.is_contiguous():
            raise ValueError("tensors must be contiguous (dense row-major)")
        return ctypes.c_void_p(arg.data_ptr())
    if isinstance(arg, (bool, np.bool_)):
        return bool(arg)
    if isinstance(arg, (int, np.integer)):
        return int(arg)
    if isinstance(arg, float) and argtype is _lib.vp:
        # numeric scalars travel by pointer in Exo's ABI
        holder = ctypes.c_float(arg)
        keepalive.append(holder)
        return ctypes.cast(ctypes.pointer(holder), ctypes.c_void_p)
    raise ValueError(f"unrecognized type {type(arg)}")


_raw_stream = None  # torch._C._cuda_getCurrentRawStream where available: the stream handle without a Stream object


def _sync_stream_for(args):
    """Device tensors run on torch's current stream."""
    global _raw_stream
    for a in args:
        if _is_torch(a) and a.is_cuda:
            if _raw_stream is None:
                import torch

                fast = getattr(torch._C, "_cuda_getCurrentRawStream", None)
                _raw_stream = fast if fast is not None else (lambda i: torch.cuda.current_stream(i).cuda_stream)
            return _raw_stream(a.device.index)
    return None


_last_default_stream = threading.local()  # what this thread last installed as the library's default stream


class ProcWrapper:
    def __init__(self, dll, name):
        self._fn = getattr(dll, name)
        self._dll = dll
        self._name = name
        self._argtypes = _lib.PROTOTYPES[name]

    def __call__(self, *args, **kwargs):
        if kwargs:
            raise ValueError("cannot call with kwargs")
        if len(args) != len(self._argtypes):
            raise TypeError(f"{self._name} takes {len(self._argtypes)} arguments ({len(args)} given)")
        stream = _sync_stream_for(args)
        keepalive = []  # per call, so concurrent callers cannot free each other's scalars
        conv = [_convert(a, t, keepalive) for a, t in zip(args, self._argtypes)]
        self._enqueue(args[0] if isinstance(args[0], Context) else None, stream, conv)
        del keepalive

    def _enqueue(self, ctx, stream, conv):
        """The call itself, on `stream` (None: no operand is on a GPU).  A context that has been closed is none."""
        if ctx is not None and ctx.handle:
            with ctx.lock:  # neither another thread's stream nor its close() may come between
                conv[0] = ctx.handle
                if stream is not None and conv[0]:
                    self._dll.exo_b200_context_set_stream(conv[0], stream)
                self._fn(*conv)
        else:
            if ctx is not None:
                conv[0] = None
            if getattr(_last_default_stream, "value", -1) != stream:
                # the library keeps the default stream per host thread; tell it only when it changes
                self._dll.exo_b200_set_default_stream(stream)
                _last_default_stream.value = stream
            self._fn(*conv)
        code = self._dll.exo_b200_last_error()
        if code != OK:
            raise ExoB200Error(code, self._dll.exo_b200_last_error_string().decode())


# element types that count as each kind of the signatures; bf16 travels as 16-bit patterns, too
_KINDS = {"bf16": ("bfloat16", "int16", "uint16"), "i8": ("int8",), "f32": ("float32",)}


class CheckedProc(ProcWrapper):
    """An entry point whose arrays and tensors are held against its signature (element type, number of elements, width
    of the rows) before the call: through raw pointers a wrong one would be read or written past its end, and a transposed
    one multiplied wrongly.  One dimension, or any number of them whose last is the row, will do.  A call of a few
    microseconds should not take four times that in its wrapper: torch tensors on a GPU go through the compiled
    ``_call``, everything else through one pass over the arguments here."""

    def __init__(self, dll, name):
        super().__init__(dll, name)
        sizes, tensors, written = _lib.SIGNATURES[name]
        self._first = 1 + sizes
        self._written = frozenset(1 + sizes + i for i in written)
        numpy_types = {k: frozenset(np.dtype(n) for n in names if n != "bfloat16") for k, names in _KINDS.items()}
        # per tensor: position, kind, numpy types, torch types (filled in when torch is there), its one or two sizes
        self._plan = [(1 + sizes + i, kind, numpy_types[kind], set(), 1 + dims[0], 1 + dims[1] if len(dims) > 1 else 0)
                      for i, (kind, _, dims) in enumerate(tensors)]
        self._torch = None  # the class torch.Tensor
        self._fast = None

    def _learn_torch(self):
        import sys

        torch = sys.modules.get("torch")
        if not hasattr(torch, "Tensor"):  # not there, or still being imported
            return
        # (torch has uint16 from 2.3 on)
        known = {kind: tuple(getattr(torch, n) for n in names if hasattr(torch, n)) for kind, names in _KINDS.items()}
        for _, kind, _, types, _, _ in self._plan:
            types.update(known[kind])
        self._torch = torch.Tensor
        current = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        if _call is not None and current is not None and isinstance(self._dll, ctypes.CDLL):
            address = lambda f: ctypes.cast(f, ctypes.c_void_p).value
            _call.setup(torch.Tensor, torch.nn.Parameter, tuple(known.values()), current, _last_default_stream,
                        address(self._dll.exo_b200_set_default_stream), address(self._dll.exo_b200_last_error))
            kinds = list(_KINDS)
            self._fast = _call.plan(address(self._fn), self._first - 1,
                                    tuple((kinds.index(kind), d0, d1) for _, kind, _, _, d0, d1 in self._plan))

    def _refuse(self, at, kind, a, have, count, width):
        name = f"{self._name}: operand {at - self._first + 1}"
        if have is None:
            raise ValueError(f"{name}: unrecognized type {type(a)}")
        if have != count:
            raise ValueError(f"{name} has {have} elements, not {count}")
        if width is not None and len(a.shape) > 1 and a.shape[-1] != width:
            raise ValueError(f"{name} has rows of {a.shape[-1]} elements, not {width}")
        if not (a.flags["C_CONTIGUOUS"] if isinstance(a, np.ndarray) else a.is_contiguous()):
            raise ValueError(f"{name} must be contiguous (dense row-major)")
        raise ValueError(f"{name} holds {a.dtype}, not {kind}")

    def __call__(self, *args, **kwargs):
        if self._fast is not None and not kwargs:
            code = _call.call(self._fast, args)
            if code == OK:
                return
            if code > OK:
                raise ExoB200Error(code, self._dll.exo_b200_last_error_string().decode())
        if kwargs:
            raise ValueError("cannot call with kwargs")
        if len(args) != len(self._argtypes):
            raise TypeError(f"{self._name} takes {len(self._argtypes)} arguments ({len(args)} given)")
        if self._torch is None:
            self._learn_torch()
        Tensor = self._torch
        conv = list(args)
        for i in range(1, self._first):
            if type(conv[i]) is not int:
                conv[i] = operator.index(conv[i])
            if not -1 << 63 <= conv[i] < 1 << 63:  # ctypes would pass its low 64 bits
                raise ValueError(f"{self._name}: argument {i} is out of range")
        stream = None
        for at, kind, numpy_types, torch_types, d0, d1 in self._plan:
            a = conv[at]
            if a is None:
                continue  # a NULL that the entry point does not take is its own refusal
            width = conv[d1] if d1 else None
            count = conv[d0] * width if d1 else conv[d0]
            if Tensor is not None and isinstance(a, Tensor):
                if (a.dtype not in torch_types or a.numel() != count or not a.is_contiguous()
                        or d1 and a.dim() > 1 and a.shape[-1] != width):
                    self._refuse(at, kind, a, a.numel(), count, width)
                if a.is_cuda and stream is None:
                    stream = _sync_stream_for((a,))
                conv[at] = a.data_ptr()
                if not conv[at] and count:  # a meta tensor, which would pass for an operand that is left out
                    raise ValueError(f"{self._name}: operand {at - self._first + 1} has no memory ({a.device})")
            elif isinstance(a, np.ndarray):
                if (a.dtype not in numpy_types or a.size != count or not a.flags["C_CONTIGUOUS"]
                        or d1 and a.ndim > 1 and a.shape[-1] != width):
                    self._refuse(at, kind, a, a.size, count, width)
                if at in self._written and not a.flags.writeable:
                    raise ValueError(f"{self._name}: operand {at - self._first + 1} is written, and the array is read-only")
                conv[at] = a.ctypes.data
            else:
                self._refuse(at, kind, a, None, count, width)
        ctx = args[0]
        if ctx is not None and not isinstance(ctx, Context):
            raise ValueError(f"unrecognized type {type(ctx)}")
        self._enqueue(ctx, stream, conv)


class Library:
    """``lib.<proc>(ctxt, ...)`` for every entry point of include/exo_b200.h."""

    def __init__(self):
        self.dll = _lib.load()

    def __getattr__(self, item):
        if item in _lib.PROTOTYPES:
            w = (CheckedProc if item in _lib.SIGNATURES else ProcWrapper)(self.dll, item)
            setattr(self, item, w)
            return w
        raise AttributeError(item)

    def synchronize(self, ctx: "Context | None" = None) -> None:
        code = self.dll.exo_b200_synchronize(ctx.handle if ctx else None)
        if code != OK:
            raise ExoB200Error(code, self.dll.exo_b200_last_error_string().decode())

    def trim(self, ctx: "Context | None" = None) -> None:
        """Gives the memory that finished calls have left with the context back to the device
        (exo_b200_context_trim)."""
        self.dll.exo_b200_context_trim(ctx.handle if ctx else None)
        code = self.dll.exo_b200_last_error()
        if code != OK:
            raise ExoB200Error(code, self.dll.exo_b200_last_error_string().decode())

    def version(self) -> str:
        return self.dll.exo_b200_version().decode()


class Context:
    """An explicit context: device, stream and SGEMM arithmetic path."""

    handle = None

    def __init__(self, device: int = -1, stream: int | None = None, sgemm_path: int = SGEMM_FFMA):
        self.lock = threading.RLock()  # held while a thread sets the stream and makes its call (a finaliser may call, too)
        self._dll = _lib.load()
        self.handle = self._dll.exo_b200_context_create(device, stream)
        if not self.handle:
            raise ExoB200Error(self._dll.exo_b200_last_error(),
                               self._dll.exo_b200_last_error_string().decode())
        self._dll.exo_b200_context_set_sgemm_path(self.handle, sgemm_path)

    def close(self):
        if self.handle:
            with self.lock:
                handle, self.handle = self.handle, None
                if handle:
                    self._dll.exo_b200_context_destroy(handle)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


_library = None


def library() -> Library:
    global _library
    if _library is None:
        _library = Library()
    return _library
