"""What the ctypes bindings of the libraries share: loading one once with its
signatures and struct layouts checked, structs filled in one pack, and the checks
of tensors that every call makes."""

from __future__ import annotations

import ctypes
import struct
import threading
from pathlib import Path

import torch  # noqa: F401  (must be loaded before the HIP library)

from ._lib import KrkError

P, I64, INT, F32, SIZE = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
_CODES = {P: "P", I64: "q", INT: "i", F32: "f"}
_ERR_HIP = -5


def _format(cls) -> str:
    return "".join(_format(t) if issubclass(t, ctypes.Structure) else _CODES[t] for _, t in cls._fields_)


def packer(cls):
    """The struct's layout for ``pack``: its fields in order, nested structs
    flattened.  One call fills it, where setting a ctypes field costs as much as
    reading a tensor's pointer."""
    s = struct.Struct("@" + _format(cls) + "0P")
    if s.size != ctypes.sizeof(cls):
        raise ImportError(f"{cls.__name__}: packed {s.size} bytes, laid out {ctypes.sizeof(cls)}")
    return s.pack


class Library:
    """A library of this package: ``lib.load()`` gives the functions of
    ``signatures`` (name -> (restype, argtypes)); names start with ``prefix``."""

    def __init__(self, path: Path, prefix: str, abi: int, structs: tuple, signatures: dict):
        self.path, self.prefix, self.abi, self.structs, self.signatures = path, prefix, abi, structs, signatures
        self._lib = None
        self._lock = threading.Lock()

    def load(self) -> ctypes.CDLL:
        """Load (once) and return the library.  Raises ImportError if it is not built."""
        if self._lib is not None:
            return self._lib
        with self._lock:
            if self._lib is None:
                if not self.path.exists():
                    raise ImportError(
                        f"{self.path} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
                        "or `python kernel-rush-kawk_amd/build_lib.py` (there is no fallback)")
                lib = ctypes.CDLL(str(self.path))
                for name, (res, args) in self.signatures.items():
                    fn = getattr(lib, name)
                    fn.restype = res
                    fn.argtypes = args
                abi = getattr(lib, self.prefix + "abi_version")()
                size = getattr(lib, self.prefix + "struct_size")
                sizes, mine = [size(i) for i in range(len(self.structs))], [ctypes.sizeof(s) for s in self.structs]
                if abi != self.abi or sizes != mine:
                    raise ImportError(f"{self.path}: ABI version {abi} with structs of {sizes} bytes; this binding expects "
                                      f"version {self.abi} and {mine} (rebuild the library or update the binding)")
                self._lib = lib
        return self._lib

    def check(self, rc: int) -> None:
        """Raise for a non-zero return code: ValueError for argument errors, KrkError for runtime errors."""
        if rc == 0:
            return
        msg = getattr(self.load(), self.prefix + "last_error")().decode(errors="replace")
        if rc == _ERR_HIP:
            raise KrkError(rc, msg)
        raise ValueError(f"krk error {rc}: {msg}")

    def launch(self, fn, index: int, *args) -> None:
        """``fn(*args, stream)`` on GPU ``index`` and torch's current stream there."""
        stream = _raw_stream(index)
        if _current() == index:
            rc = fn(*args, stream)
        else:
            with torch.cuda.device(index):
                rc = fn(*args, stream)
        if rc:
            self.check(rc)


_raw_stream = torch._C._cuda_getCurrentRawStream
_current = torch._C._cuda_getDevice


def ints(**sizes) -> None:
    """Sizes that fit the structs' ints (which would take others modulo 2^32)."""
    for name, n in sizes.items():
        if not isinstance(n, int) or not -1 << 31 <= n < 1 << 31:
            raise ValueError(f"{name} must be an int of 32 bits, got {n!r}")


def index_of(name: str, t: torch.Tensor) -> int:
    """The GPU that a call's first operand is on."""
    if isinstance(t, torch.Tensor):
        index = t.get_device()
        if index >= 0 and t.is_cuda:
            return index
        raise ValueError(f"{name} must be a GPU tensor, got device {t.device}")
    raise ValueError(f"{name} must be a torch.Tensor")


def _refuse(name: str, t, index: int, dtype: torch.dtype, shape: tuple, layout: str):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch.Tensor")
    if t.get_device() != index or not t.is_cuda:
        raise ValueError(f"{name} must be on the operands' GPU, got {t.device}")
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError(f"{name} must be {dtype} of shape {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
    raise ValueError(f"{name}: {layout}, got strides {t.stride()}")


def rows(name: str, t: torch.Tensor, index: int, shape: tuple, dtype: torch.dtype = torch.bfloat16) -> tuple:
    """Address and row stride of a [rows, columns] tensor."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == index:
        row, one = t.stride()
        if one == 1 or t.shape[1] == 1:
            return t.data_ptr(), row
    _refuse(name, t, index, dtype, shape, "rows must be contiguous")


def blocks(name: str, t: torch.Tensor, index: int, shape: tuple) -> tuple:
    """Address and outer strides of a bf16 tensor whose last dimension is contiguous."""
    if isinstance(t, torch.Tensor) and t.dtype is torch.bfloat16 and t.shape == shape and t.get_device() == index:
        *outer, one = t.stride()
        if one == 1:
            return t.data_ptr(), *outer
    _refuse(name, t, index, torch.bfloat16, shape, "the last dimension must be contiguous")


def plain(name: str, t: torch.Tensor, index: int, dtype: torch.dtype, shape: tuple) -> int:
    """The address of a contiguous tensor of this type and shape."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous():
        return t.data_ptr()
    _refuse(name, t, index, dtype, shape, "it must be contiguous")


class Owner:
    """An object with GPU memory of its own (``tensors``) that calls on any stream
    use.  It is not given to others before those streams are through with it, also
    where the object goes first.  (Of a captured graph only its owner knows when it
    runs last.)"""

    def __init__(self, device, tensors: tuple):
        self.device = torch.device(device)
        self._tensors = tensors
        self._streams: set = set()
        if self.device.type == "cuda" and tensors:  # filled on this stream, used on others
            torch.cuda.current_stream(self.device).synchronize()

    def outlive(self, index: int) -> None:
        stream = _raw_stream(index)
        if stream not in self._streams and not torch.cuda.is_current_stream_capturing():
            now = torch.cuda.current_stream(index)
            for t in self._tensors:
                t.record_stream(now)
            self._streams.add(stream)


def refuse_capture(device) -> None:
    """Memory of an object is filled, and waited for, when it is built."""
    if torch.device(device).type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("an object's memory is filled when it is built: build it before the capture")
