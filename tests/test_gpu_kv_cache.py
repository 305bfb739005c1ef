"""KvCache.write and KvCache.read: what the cache holds is the package's host
quantiser's result, bit for bit, and nothing else moves."""
import ctypes as C

import numpy as np
import pytest

from dotllm_amd import Q4_0, Q8_0, DeviceArray, KvCache
from dotllm_amd._lib import lib
from dotllm_amd.backend import HipBackend, _call
from tests.kv_reference import held

pytestmark = pytest.mark.gpu

TYPES = [(Q8_0, Q8_0), (Q4_0, Q4_0), (Q8_0, Q4_0), (Q4_0, Q8_0)]
SENTINEL = -77.0


def _i32(be, v):
    return DeviceArray.of(be, v, np.int32)


def read_all(be, cache):
    """Every position of every slot, [slots, capacity, kv_heads, head_dim]."""
    shape = (cache.slots, cache.capacity, cache.kv_heads, cache.head_dim)
    k, v = DeviceArray(be, shape), DeviceArray(be, shape)
    batch = cache.batch(cache.capacity, _i32(be, np.arange(cache.slots)), _i32(be, np.zeros(cache.slots)))
    cache.read(k, v, batch)
    return k.get(), v.get()


def rows_of(rng, *shape):
    x = rng.standard_normal(shape).astype(np.float32)
    return x * np.exp(rng.normal(size=shape[:-1] + (1,)) * 2).astype(np.float32)   # rows of very different size


def check_write(be, cache, k, v, slots, starts, counts, want_k, want_v):
    n, tokens = k.shape[:2]
    batch = cache.batch(tokens, _i32(be, slots), _i32(be, starts), None if counts is None else _i32(be, counts))
    cache.write(DeviceArray.of(be, k), DeviceArray.of(be, v), batch)
    hk, hv = held(k, cache.k_type), held(v, cache.v_type)
    for b in range(n):
        count = tokens if counts is None else max(0, min(tokens, counts[b]))
        if not 0 <= slots[b] < cache.slots:
            continue
        for i in range(count):
            p = starts[b] + i
            if 0 <= p < cache.capacity:
                want_k[slots[b], p], want_v[slots[b], p] = hk[b, i], hv[b, i]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("head_dim,kv_heads", [(64, 3), (96, 1), (128, 2), (256, 1)])
def test_rows_are_the_host_quantisers(hip, types, head_dim, kv_heads):
    rng = np.random.default_rng(head_dim + kv_heads)
    with KvCache(hip, 4, kv_heads, head_dim, 75, *types) as cache:
        assert all(not x.any() for x in read_all(hip, cache))
        want_k = np.zeros((4, 75, kv_heads, head_dim))
        want_v = np.zeros_like(want_k)
        # single tokens, a run across record borders, ragged runs, then rows that leave the slot at either end
        for tokens, slots, starts, counts in [(1, [2], [31], None), (1, [2], [32], None), (70, [1], [3], None),
                                              (33, [0, 3, 2], [1, 30, 40], [33, 5, 0]),
                                              (40, [3, 1], [60, -7], [40, 9]), (2, [3, 0], [74, 2], [2, 1])]:
            k = rows_of(rng, len(slots), tokens, kv_heads, head_dim)
            v = rows_of(rng, len(slots), tokens, kv_heads, head_dim)
            check_write(hip, cache, k, v, slots, starts, counts, want_k, want_v)
            got_k, got_v = read_all(hip, cache)
            assert np.array_equal(got_k, want_k) and np.array_equal(got_v, want_v)


@pytest.mark.parametrize("types", TYPES[:2])
def test_special_rows(hip, types):
    """Zeros, one value alone, equal magnitudes of either sign, subnormal scales and borders between integers; then
    what the host quantiser has no number for: scales past fp16's largest are held as it, NaN as 0."""
    hd = 64
    x = np.zeros((1, 9, 1, hd), dtype=np.float32)
    x[0, 1, 0, 5] = -3.0
    x[0, 2, 0, :] = np.where(np.arange(hd) % 3 == 0, -2.0, 2.0)
    x[0, 3, 0, :] = np.linspace(-1e-6, 1e-6, hd)
    x[0, 4, 0, :] = np.linspace(-3e-8, 2e-8, hd)
    x[0, 5, 0, :32] = np.arange(32) - 15.5          # halves of the step 15.5 / 127 and others
    x[0, 5, 0, 0] = 127.0
    x[0, 5, 0, 32:] = np.arange(32) + 0.5
    x[0, 5, 0, 32] = -8.0 if types[0] == Q4_0 else 127.0
    x[0, 6, 0, :] = np.linspace(-6e4, 6e4, hd)
    x[0, 7, 0, :] = np.nextafter(np.float32(0.5), np.float32(0)) * np.arange(hd)
    x[0, 8, 0, :] = -np.linspace(0, 1, hd) ** 8
    with KvCache(hip, 1, 1, hd, 32, *types) as cache:
        want_k, want_v = np.zeros((1, 32, 1, hd)), np.zeros((1, 32, 1, hd))
        check_write(hip, cache, x, x, [0], [4], None, want_k, want_v)
        got_k, got_v = read_all(hip, cache)
        assert np.array_equal(got_k, want_k) and np.array_equal(got_v, want_v)
        y = np.ones((1, 4, 1, hd), dtype=np.float32)
        y[0, 0, 0, 3], y[0, 0, 0, 40] = np.inf, -np.inf
        y[0, 1, 0, 7] = np.nan
        y[0, 2, 0, 9] = 3e38
        y[0, 3, 0, :] = np.nan
        cache.write(DeviceArray.of(hip, y), DeviceArray.of(hip, y), cache.batch(4, _i32(hip, [0]), _i32(hip, [20])))
        got = read_all(hip, cache)
        for g in got:
            g = g[0, 20:24, 0]
            assert np.isfinite(g).all()
            assert abs(g[0, 3]) >= 65504.0 * 7 and g[0, 40] <= -65504.0 * 7
            assert g[1, 7] == 0.0 and np.allclose(np.delete(g[1], 7), 1.0, atol=1e-3)
            assert g[2, 9] >= 65504.0 * 7 and not g[3].any()


def test_the_later_of_two_rows_for_one_position_is_kept(hip):
    rng = np.random.default_rng(3)
    with KvCache(hip, 2, 2, 64, 80, Q4_0, Q8_0) as cache:
        want_k, want_v = np.zeros((2, 80, 2, 64)), np.zeros((2, 80, 2, 64))
        for _ in range(3):
            k, v = rows_of(rng, 5, 40, 2, 64), rows_of(rng, 5, 40, 2, 64)
            check_write(hip, cache, k, v, [1, 0, 1, 1, 0], [2, 0, 2, 30, 39], [40, 40, 20, 40, 1], want_k, want_v)
            got_k, got_v = read_all(hip, cache)
            assert np.array_equal(got_k, want_k) and np.array_equal(got_v, want_v)


def test_read_leaves_other_rows(hip):
    rng = np.random.default_rng(5)
    with KvCache(hip, 3, 2, 96, 50) as cache:
        want_k, want_v = np.zeros((3, 50, 2, 96)), np.zeros((3, 50, 2, 96))
        k = rows_of(rng, 3, 50, 2, 96)
        check_write(hip, cache, k, k, [0, 1, 2], [0, 0, 0], None, want_k, want_v)
        out = DeviceArray.of(hip, np.full((5, 7, 2, 96), SENTINEL, np.float32))
        out_v = DeviceArray.of(hip, np.full((5, 7, 2, 96), SENTINEL, np.float32))
        slots, starts, counts = [1, 7, 2, -1, 0], [46, 0, -3, 0, 2 ** 31 - 1], [7, 7, 6, 3, 7]
        cache.read(out, out_v, cache.batch(7, _i32(hip, slots), _i32(hip, starts), _i32(hip, counts)))
        want = np.full((5, 7, 2, 96), SENTINEL)
        want[0, :4] = want_k[1, 46:50]
        want[2, 3:6] = want_k[2, 0:3]
        assert np.array_equal(out.get(), want)
        assert np.array_equal(out_v.get(), want)


def test_rows_of_a_fused_projection(hip):
    """k and v as row ranges of wider rows, read back into ranges of others: strides through the C ABI."""
    rng = np.random.default_rng(1)
    wide = rng.standard_normal((2, 9, 10, 64)).astype(np.float32)
    dev, out = DeviceArray.of(hip, wide), DeviceArray.of(hip, np.full(wide.shape, SENTINEL, np.float32))
    with KvCache(hip, 2, 3, 64, 40) as cache:
        batch = cache.batch(9, _i32(hip, [0, 1]), _i32(hip, [1, 20]))
        at = lambda x, head: x.data_ptr() + head * 64 * 4   # noqa: E731
        call = lib().llmdot_hip_kv_cache_write
        _call(call(cache.handle, at(dev, 4), 640, at(dev, 7), 640, C.byref(batch.struct)))
        _call(lib().llmdot_hip_kv_cache_read(cache.handle, at(out, 4), 640, at(out, 7), 640, C.byref(batch.struct)))
        got = out.get()
        assert (got[:, :, :4] == SENTINEL).all()
        assert np.array_equal(got[:, :, 4:7], held(wide[:, :, 4:7], Q8_0))
        assert np.array_equal(got[:, :, 7:], held(wide[:, :, 7:], Q8_0))
        for kp, ks in ((at(dev, 4), 639), (at(dev, 4), 188), (at(dev, 4), -640), (at(dev, 4) + 4, 640), (None, 640)):
            with pytest.raises(ValueError):
                _call(call(cache.handle, kp, ks, at(dev, 7), 640, C.byref(batch.struct)))


def test_positions_past_four_gigabytes(hip):
    """Offsets that pass 32 bits, in bytes and in elements."""
    rng = np.random.default_rng(11)
    cap = 1 << 20
    with KvCache(hip, 5, 8, 128, cap) as cache:   # 5.7 GB of keys
        slots, starts = [4, 0, 4, 2], [cap - 3, 0, 5, cap - 40]
        k, v = rows_of(rng, 4, 3, 8, 128), rows_of(rng, 4, 3, 8, 128)
        batch = cache.batch(3, _i32(hip, slots), _i32(hip, starts))
        cache.write(DeviceArray.of(hip, k), DeviceArray.of(hip, v), batch)
        ko, vo = DeviceArray(hip, k.shape), DeviceArray(hip, v.shape)
        cache.read(ko, vo, batch)
        assert np.array_equal(ko.get(), held(k, Q8_0)) and np.array_equal(vo.get(), held(v, Q8_0))


def test_refusals(hip):
    with pytest.raises(NotImplementedError):
        KvCache(hip, 1, 1, 80, 16)
    with pytest.raises(NotImplementedError):
        KvCache(hip, 1, 1, 64, 16, k_type=14)
    for bad in ((0, 1, 64, 16), (1, 0, 64, 16), (1, 1, 64, 0), (1, 1, -64, 16)):
        with pytest.raises(ValueError):
            KvCache(hip, *bad)
    cache = KvCache(hip, 1, 2, 64, 16)
    k = DeviceArray(hip, (1, 2, 2, 64))
    one = _i32(hip, [0])
    with pytest.raises(ValueError):
        cache.batch(1, one, _i32(hip, [0, 1]))
    with pytest.raises(ValueError):
        cache.batch(1, one, DeviceArray(hip, (1,)))
    batch = cache.batch(2, one, one)
    cache.write(k, k, batch)
    for bad in (DeviceArray(hip, (1, 2, 2, 32)), np.zeros((1, 2, 2, 64), np.float32), _i32(hip, np.zeros((1, 2, 2, 64)))):
        with pytest.raises(ValueError):
            cache.write(k, bad, batch)
        with pytest.raises(ValueError):
            cache.read(bad, k, batch)
    with pytest.raises(ValueError):
        cache.write(k, k, cache.batch(-2, one, one))
    empty = cache.batch(0, one, one)
    cache.write(DeviceArray(hip, (1, 0, 2, 64)), DeviceArray(hip, (1, 0, 2, 64)), empty)
    cache.dispose()
    with pytest.raises(ValueError):
        cache.write(k, k, batch)


def test_a_context_outlives_its_caches():
    be = HipBackend(0)
    cache = KvCache(be, 1, 1, 64, 16)
    x = DeviceArray(be, (1, 1, 1, 64))
    one = _i32(be, [0])
    batch = cache.batch(1, one, one)
    x.free()
    one.free()
    be.dispose()
    cache.dispose()
    del batch
