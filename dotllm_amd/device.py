"""Arrays in device memory for the operators that take device addresses.

Such an operator takes a :class:`DeviceArray` or any other contiguous array in
HBM that says where it lies: a torch tensor, or an object with
``__cuda_array_interface__``.  Calls run on the backend's stream
(:attr:`HipBackend.stream`); an array that another stream writes or reads is
ordered by the caller with events, or by synchronising.  torch brings a HIP
runtime of its own: a program that uses both imports torch before it creates a
backend, so that they share one.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from ._lib import call, lib, ptr

_TYPES = {"float32": "<f4", "int32": "<i4"}


class DeviceArray:
    """Zeroed memory of a backend's device, freed with the array."""

    def __init__(self, backend: "HipBackend", shape, dtype="float32"):
        self.backend = backend
        self.shape = tuple(int(n) for n in (shape if hasattr(shape, "__len__") else (shape,)))
        self.dtype = np.dtype(dtype)
        if any(n < 0 for n in self.shape):
            raise ValueError(f"negative size in {self.shape}")
        self.size = int(np.prod(self.shape, dtype=np.int64))
        self.nbytes = self.size * self.dtype.itemsize
        self._p = C.c_void_p()
        call(lib().llmdot_hip_device_alloc(backend.handle, max(self.nbytes, 16), C.byref(self._p)))

    @classmethod
    def of(cls, backend: "HipBackend", values, dtype=None) -> "DeviceArray":
        """A copy of host values."""
        a = np.ascontiguousarray(values, dtype=dtype)
        out = cls(backend, a.shape, a.dtype)
        out.put(a)
        return out

    def put(self, values) -> None:
        """Copies host values in, in the order of the backend's stream."""
        a = np.ascontiguousarray(values, dtype=self.dtype)
        if a.size != self.size:
            raise ValueError(f"{a.size} values for an array of {self.size}")
        if a.nbytes:
            call(lib().llmdot_hip_memcpy_h2d(self.backend.handle, self._p, ptr(a), a.nbytes))

    def get(self) -> np.ndarray:
        """The values on the host, after everything the backend's stream holds."""
        a = np.empty(self.shape, dtype=self.dtype)
        if a.nbytes:
            call(lib().llmdot_hip_memcpy_d2h(self.backend.handle, ptr(a), self._p, a.nbytes))
        return a

    @property
    def device(self) -> "Place":
        return self.backend.place

    def data_ptr(self) -> int:
        return self._p.value

    def is_contiguous(self) -> bool:
        return True

    @property
    def __cuda_array_interface__(self) -> dict:
        return {"shape": self.shape, "typestr": self.dtype.str, "data": (self._p.value, False), "version": 2}

    def free(self) -> None:
        if self._p:
            if self.backend.handle:   # a disposed backend cannot be waited for
                lib().llmdot_hip_device_free(self.backend.handle, self._p)
            self._p = C.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


_NAMES = {"float32": ("float32", "torch.float32"), "int32": ("int32", "torch.int32")}
_KNOWN = {"float32": set(), "int32": set()}   # types of other libraries that go by these names


def _typed(dtype, name: str) -> bool:
    if dtype in _KNOWN[name]:
        return True
    if str(dtype) in _NAMES[name]:
        _KNOWN[name].add(dtype)
        return True
    return False


def address(a, name: str, dtype: str, shape: tuple, device: int) -> int:
    """The address of a contiguous device array of the given type and shape."""
    where = getattr(a, "data_ptr", None)
    if where is not None:
        if a.device.index != device or a.shape != shape or not _typed(a.dtype, dtype) or not a.is_contiguous():
            _refuse(a, name, dtype, shape, device)
        return where()
    face = getattr(a, "__cuda_array_interface__", None)
    if face is None:
        raise ValueError(f"{name} must be an array in device memory")
    if face["typestr"] != _TYPES[dtype]:
        raise ValueError(f"{name} must be {dtype}, not {face['typestr']}")
    if tuple(face["shape"]) != shape:
        raise ValueError(f"{name} must have shape {shape}, not {tuple(face['shape'])}")
    strides = face.get("strides")
    if strides is not None:
        want, step = [], np.dtype(dtype).itemsize
        for n in reversed(shape):
            want.insert(0, step)
            step *= n
        if any(s != w and n > 1 for s, w, n in zip(strides, want, shape)):
            raise ValueError(f"{name} must be contiguous")
    return face["data"][0]


def _refuse(a, name: str, dtype: str, shape: tuple, device: int) -> None:
    if a.device.index != device:   # host arrays have no index
        raise ValueError(f"{name} is on {a.device}, not on device {device}")
    if tuple(a.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, not {tuple(a.shape)}")
    if not _typed(a.dtype, dtype):
        raise ValueError(f"{name} must be {dtype}, not {a.dtype}")
    raise ValueError(f"{name} must be contiguous")


def workspace_room(a, device: int) -> tuple:
    """Address and bytes of a workspace."""
    if a.device.index != device:
        raise ValueError(f"the workspace is on {a.device}, not on device {device}")
    if not a.is_contiguous():
        raise ValueError("the workspace must be contiguous")
    return a.data_ptr(), a.nbytes


def rows(a, name: str, shape: tuple, device: int) -> tuple:
    """Address and row stride (floats) of a float32 array [batch, tokens, heads, head_dim] whose
    rows are whole and equally far apart: contiguous, or a slice of wider rows (a fused projection's)."""
    stride = getattr(a, "stride", None)
    if stride is None:
        return address(a, name, "float32", shape, device), 0
    if a.device.index != device or a.shape != shape or not (a.dtype in _KNOWN["float32"] or _typed(a.dtype, "float32")):
        _refuse(a, name, "float32", shape, device)
    if a.is_contiguous():
        return a.data_ptr(), 0
    b, t, h, d = shape
    sb, st, sh, sd = stride()
    if 0 in shape or sd != 1 or (h > 1 and sh != d):
        raise ValueError(f"{name}'s rows must be contiguous")
    step = st if t > 1 else sb if b > 1 else 0
    if b > 1 and t > 1 and sb != t * st or b * t > 1 and step <= 0:   # the same row again: 0 would say packed
        raise ValueError(f"{name}'s rows must be equally far apart")
    return a.data_ptr(), step
