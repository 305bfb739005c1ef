"""KvCache: a quantised KV cache in device memory, and attention over it.

The cache holds `slots` sequences of `capacity` positions in the block formats
Q8_0 or Q4_0 (keys and values apart), quantised as rows are written: a quarter
or an eighth of the reference's fp32 cache
(src/Llmdot.Core/Inference/KvCache.cs), which holds one sequence.  A serving
loop writes the new tokens' keys and values and attends with their queries:

    cache = KvCache(backend, slots=8, kv_heads=8, head_dim=128, capacity=4096)
    batch = cache.batch(1, slots, starts)          # device int32 arrays, updated in place
    cache.write(k, v, batch)                       # [sequences, 1, 8, 128] float32
    cache.attention(q, out, batch, workspace=ws)   # [sequences, 1, 32, 128] float32

Everything runs on the backend's stream and allocates nothing, so a loop's step
can be captured into a HIP graph.  See include/llmdot_hip_cache.h.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import Q8_0, call, lib
from .backend import HipBackend
from .device import DeviceArray, address, rows, workspace_room


class TokenBatch:
    """The tokens of a call (:meth:`KvCache.batch`); keeps its arrays alive."""

    def __init__(self, sequences: int, tokens: int, arrays: tuple, addresses: tuple, device: int):
        self.sequences, self.tokens, self._arrays, self.device = sequences, tokens, arrays, device
        self.struct = _lib.TokenBatch(sequences, tokens, *addresses)
        self.ref = C.byref(self.struct)


class KvCache:
    def __init__(self, backend: HipBackend, slots: int, kv_heads: int, head_dim: int, capacity: int,
                 k_type: int = Q8_0, v_type: int = Q8_0):
        self._c = C.c_void_p()
        self.backend = backend
        self.slots, self.kv_heads, self.head_dim, self.capacity = slots, kv_heads, head_dim, capacity
        self.k_type, self.v_type = k_type, v_type
        d = _lib.KvCacheDesc(slots, kv_heads, head_dim, capacity, k_type, v_type)
        self._lib = lib()
        call(self._lib.llmdot_hip_kv_cache_create(backend.handle, C.byref(d), C.byref(self._c)))

    def dispose(self) -> None:
        if self._c:
            lib().llmdot_hip_kv_cache_destroy(self._c)
            self._c = C.c_void_p()

    close = dispose

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.dispose()

    def __del__(self):
        try:
            self.dispose()
        except Exception:
            pass

    @property
    def handle(self) -> C.c_void_p:
        if not self._c:
            raise ValueError("the cache has been disposed")
        return self._c

    def batch(self, tokens: int, slots, starts, counts=None) -> TokenBatch:
        """Sequences of `tokens` rows each: sequence b's first counts[b] rows (all, without
        counts) are positions starts[b] .. of slot slots[b].  Device int32 arrays, one value per
        sequence, read when a call runs: a loop updates them in place."""
        n = int(slots.shape[0])
        dev = self.backend.device
        arrays = (slots, starts) + (() if counts is None else (counts,))
        at = [address(a, name, "int32", (n,), dev) for a, name in zip(arrays, ("slots", "starts", "counts"))]
        return TokenBatch(n, int(tokens), arrays, (*at, *([None] * (3 - len(at)))), dev)

    def _device(self, batch: TokenBatch) -> int:
        dev = self.backend.device
        if batch.device != dev:
            raise ValueError(f"the batch is on device {batch.device}, the cache on device {dev}")
        return dev

    def write(self, k, v, batch: TokenBatch) -> None:
        """Quantises k and v [sequences, tokens, kv_heads, head_dim] into the cache."""
        dev, shape = self._device(batch), (batch.sequences, batch.tokens, self.kv_heads, self.head_dim)
        kp, ks = rows(k, "k", shape, dev)
        vp, vs = rows(v, "v", shape, dev)
        call(self._lib.llmdot_hip_kv_cache_write(self.handle, kp, ks, vp, vs, batch.ref))

    def read(self, k_out, v_out, batch: TokenBatch) -> None:
        """What the cache holds at the batch's positions, as fp32; other rows stay as they are."""
        dev, shape = self._device(batch), (batch.sequences, batch.tokens, self.kv_heads, self.head_dim)
        kp, ks = rows(k_out, "k_out", shape, dev)
        vp, vs = rows(v_out, "v_out", shape, dev)
        call(self._lib.llmdot_hip_kv_cache_read(self.handle, kp, ks, vp, vs, batch.ref))

    def attention_workspace(self, heads: int, sequences: int, tokens: int, prefix: bool = False) -> DeviceArray:
        """Device memory that suffices for attention calls of that size."""
        n = C.c_size_t(0)
        call(lib().llmdot_hip_kv_cache_attention_workspace(self.handle, heads, sequences, tokens, int(prefix),
                                                            C.byref(n)))
        return DeviceArray(self.backend, (n.value,), "uint8")

    def attention(self, q, out, batch: TokenBatch, *, workspace: DeviceArray, prefix: "KvCache | None" = None,
                  prefix_slot: int = 0, prefix_len: int = 0, window: int = 0, scale: float = 0.0) -> None:
        """out = softmax(scale q k) v over each token's positions, q and out
        [sequences, tokens, heads, head_dim].  Rows 0 .. prefix_len - 1 of slot `prefix_slot` of
        `prefix` come before every sequence's own; window > 0 keeps the last `window` positions;
        scale 0 is 1 / sqrt(head_dim).  Rows past a sequence's count stay as they are."""
        dev = self._device(batch)
        shape = (batch.sequences, batch.tokens, q.shape[2] if len(q.shape) == 4 else 0, self.head_dim)
        qp, qs = rows(q, "q", shape, dev)
        op, os_ = rows(out, "out", shape, dev)
        wp, room = workspace_room(workspace, dev)
        opt = _lib.Attention(shape[2], window, scale, prefix.handle if prefix is not None else None, prefix_slot,
                             prefix_len, qs, os_)
        call(self._lib.llmdot_hip_kv_cache_attention(self.handle, qp, op, batch.ref, C.byref(opt), wp, room))
