"""The operators over device memory, as far as they go without a device: exports,
bindings, refusals that need no context, and the checks of array arguments."""
import ctypes as C
import os
import re

import numpy as np
import pytest

from dotllm_amd import _lib
from dotllm_amd.device import address, rows, workspace_room
from dotllm_amd.kvcache import KvCache, TokenBatch
from tests.kv_reference import attend, held, verify

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _header():
    text = open(os.path.join(ROOT, "include", "llmdot_hip_cache.h")).read()
    return re.sub(r"/\*.*?\*/", "", text, flags=re.S)


def declared():
    return {m.group(1): m.group(2).count(",") + 1
            for m in re.finditer(r"^\s*int32_t\s+(llmdot_hip_\w+)\s*\(([^;]*?)\)\s*;", _header(), re.M | re.S)}


def test_every_declared_function_is_exported_and_bound():
    names = declared()
    assert len(names) == 9
    assert {n: len(a) for n, a in _lib.CACHE_SIGNATURES.items()} == names
    for n in names:
        assert hasattr(_lib.lib(), n)


def test_csharp_declares_every_function():
    path = os.path.join(ROOT, "dotllm_amd", "csharp", "Llmdot.Hip", "Native", "HipCacheNative.cs")
    found = {m.group(1): m.group(2).count(",") + 1
             for m in re.finditer(r"static extern int (llmdot_hip_\w+)\(([^)]*)\);", open(path).read())}
    assert found == declared()


def test_struct_sizes():
    """As a C compiler lays them out: 4-byte fields, then 8-byte aligned pointers."""
    assert C.sizeof(_lib.KvCacheDesc) == 24
    assert C.sizeof(_lib.TokenBatch) == 8 + 3 * 8
    assert C.sizeof(_lib.Attention) == 16 + 8 + 8 + 16
    assert _lib.Attention.prefix.offset == 16 and _lib.Attention.q_stride.offset == 32


def test_null_handles_are_refused():
    lib = _lib.lib()
    n = C.c_size_t(0)
    out = C.c_void_p()
    batch = _lib.TokenBatch(1, 1, None, None, None)
    for rc in (lib.llmdot_hip_stream(None, C.byref(out)),
               lib.llmdot_hip_kv_cache_create(None, C.byref(_lib.KvCacheDesc(1, 1, 64, 1, 8, 8)), C.byref(out)),
               lib.llmdot_hip_kv_cache_write(None, 16, 0, 16, 0, C.byref(batch)),
               lib.llmdot_hip_kv_cache_read(None, 16, 0, 16, 0, C.byref(batch)),
               lib.llmdot_hip_kv_cache_attention(None, 16, 16, C.byref(batch), C.byref(_lib.Attention()), None, 0),
               lib.llmdot_hip_kv_cache_attention_workspace(None, 1, 1, 1, 0, C.byref(n)),
               lib.llmdot_hip_verify_drafts(None, 16, None, 16, None, 16, 1, 1, 8, 1.0, 16, 16, None, 0),
               lib.llmdot_hip_verify_drafts_workspace(None, 1, 1, 8, C.byref(n))):
        assert rc == _lib.E_INVALID
    assert lib.llmdot_hip_kv_cache_destroy(None) == 0


class _Tensor:
    """What `rows` and `address` look at in a tensor of another owner."""

    def __init__(self, shape, strides=None, dtype="torch.float32", device="cuda", index=0):
        self.shape, self.dtype = shape, dtype
        self.device = type("D", (), dict(type=device, index=index))()
        packed = [int(np.prod(shape[i + 1:])) for i in range(len(shape))]
        self._strides = list(strides or packed)
        self._packed = self._strides == packed

    def data_ptr(self):
        return 4096

    def stride(self):
        return self._strides

    def is_contiguous(self):
        return self._packed


def test_rows():
    shape = (2, 3, 4, 64)
    assert rows(_Tensor(shape), "k", shape, 0) == (4096, 0)
    assert rows(_Tensor(shape, (3 * 640, 640, 64, 1)), "k", shape, 0) == (4096, 640)   # a slice of 10 heads' rows
    assert rows(_Tensor((1, 3, 4, 64), (9, 640, 64, 1)), "k", (1, 3, 4, 64), 0) == (4096, 640)
    assert rows(_Tensor((2, 1, 4, 64), (640, 9, 64, 1)), "k", (2, 1, 4, 64), 0) == (4096, 640)
    bad = [_Tensor(shape, (3 * 640, 640, 128, 1)), _Tensor(shape, (3 * 640, 640, 64, 2)),
           _Tensor(shape, (4 * 640, 640, 64, 1)), _Tensor(shape, (640, 1280, 64, 1)), _Tensor((2, 3, 64, 4)),
           _Tensor(shape, dtype="torch.float16"), _Tensor(shape, device="cpu", index=None), _Tensor(shape, index=1),
           _Tensor(shape, (3 * 640, 640, 64, 1), dtype="torch.float64"),
           _Tensor(shape, (3 * 640, 640, 64, 1), index=1), np.zeros(shape, np.float32), None]
    for x in bad:
        with pytest.raises(ValueError):
            rows(x, "k", shape, 0)


def test_rows_that_are_one_row_again():
    """Broadcast rows (stride 0) are no packed rows."""
    for shape, strides in (((2, 3, 4, 64), (0, 0, 64, 1)), ((1, 3, 4, 64), (768, 0, 64, 1)), ((3, 1, 4, 64), (0, 256, 64, 1))):
        with pytest.raises(ValueError):
            rows(_Tensor(shape, strides), "k", shape, 0)
    assert rows(_Tensor((1, 1, 4, 64), (0, 0, 64, 1)), "k", (1, 1, 4, 64), 0) == (4096, 0)


def test_workspace_and_batch_of_another_device():
    ok = _Tensor((64,), dtype="torch.uint8")
    ok.nbytes = 64
    assert workspace_room(ok, 0) == (4096, 64)
    for bad in (_Tensor((64,), index=1), _Tensor((64,), device="cpu", index=None), _Tensor((64,), (2,))):
        bad.nbytes = 64
        with pytest.raises(ValueError):
            workspace_room(bad, 0)
    cache = object.__new__(KvCache)   # no device is needed for what is refused before the library
    cache._c, cache.kv_heads, cache.head_dim = None, 4, 64
    cache.backend = type("B", (), dict(device=1))()
    x, batch = _Tensor((1, 1, 4, 64), index=1), TokenBatch(1, 1, (), (None, None, None), 0)
    for call in (lambda: cache.write(x, x, batch), lambda: cache.read(x, x, batch),
                 lambda: cache.attention(x, x, batch, workspace=ok)):
        with pytest.raises(ValueError, match="batch is on device 0"):
            call()


def test_address_of_an_array_interface():
    class Face:
        def __init__(self, **kw):
            self.__cuda_array_interface__ = dict(shape=(2, 5), typestr="<i4", data=(64, False), version=2, **kw)
    assert address(Face(), "slots", "int32", (2, 5), 0) == 64
    assert address(Face(strides=(20, 4)), "slots", "int32", (2, 5), 0) == 64
    for face, dtype, shape in ((Face(strides=(40, 4)), "int32", (2, 5)), (Face(), "float32", (2, 5)), (Face(), "int32", (5, 2))):
        with pytest.raises(ValueError):
            address(face, "slots", dtype, shape, 0)


def test_plain_attention_against_a_softmax_by_hand():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((2, 2, 8)), rng.standard_normal((6, 1, 8)), rng.standard_normal((6, 1, 8))
    out, tol = attend(q, k, v, 4, window=3)
    s = np.array([k[t, 0] @ q[0, 1] / np.sqrt(8) for t in (2, 3, 4)])
    w = np.exp(s) / np.exp(s).sum()
    assert np.allclose(out[0, 1], sum(w[j] * v[2 + j, 0] for j in range(3)))
    assert (tol > 0).all() and (tol < 1e-4).all()


def test_plain_verification():
    """Two tokens of probability 3/4 and 1/4; the draft model says 1/4 and 3/4."""
    target, draft = np.log(np.array([[3.0, 1.0], [3.0, 1.0]])), np.log(np.array([[1.0, 3.0]]))
    one = np.array([1], np.int32)
    assert verify(target, one, np.array([0.3, 0.7]), 1.0, draft)[1] == 1     # 0.3 * 3/4 < 1/4
    assert verify(target, one, np.array([0.4, 0.99]), 1.0, draft)[0].tolist() == [0, -1]   # only token 0 is left over
    assert verify(target, one, np.array([0.3, 0.8]), 1.0, draft)[0].tolist() == [1, 1]
    assert verify(target, np.array([0], np.int32), np.array([0.9, 0.1]), 0.0)[0].tolist() == [0, 0]


def test_held_values_are_the_quantisers():
    x = np.zeros((1, 32), np.float32)
    x[0, :3] = 127.0, -1.5, 0.49
    y = held(x, 8)
    assert y[0, :3].tolist() == [127.0, -2.0, 0.0]
