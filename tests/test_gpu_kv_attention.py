"""KvCache.attention against a plain 64-bit form over what the cache holds."""
import itertools

import numpy as np
import pytest

from dotllm_amd import Q4_0, Q8_0, DeviceArray, KvCache
from tests.kv_reference import attend, held

pytestmark = pytest.mark.gpu

SENTINEL = -77.0


def _i32(be, v):
    return DeviceArray.of(be, v, np.int32)


class Case:
    """A cache whose slots hold `lengths` positions, and what they stand for."""

    def __init__(self, be, kv_heads, head_dim, lengths, types=(Q8_0, Q8_0), prefix=0, capacity=None, seed=0,
                 k_of=None, v_of=None):
        rng = self.rng = np.random.default_rng(seed)
        self.be, self.kv_heads, self.head_dim, self.types = be, kv_heads, head_dim, types
        n, cap = len(lengths), capacity or max(max(lengths), 1)
        self.cache = KvCache(be, n, kv_heads, head_dim, cap, *types)

        def rows(m, size, change):
            x = rng.standard_normal((m, size, kv_heads, head_dim)).astype(np.float32)
            return x if change is None else change(x).astype(np.float32)

        def fill(cache, m, size):
            k, v = rows(m, size, k_of), rows(m, size, v_of)
            cache.write(DeviceArray.of(be, k), DeviceArray.of(be, v),
                        cache.batch(size, _i32(be, np.arange(m)), _i32(be, np.zeros(m))))
            return held(k, types[0]), held(v, types[1])

        self.k, self.v = fill(self.cache, n, max(max(lengths), 1))
        self.prefix, self.prefix_len = None, prefix
        if prefix:   # in the second slot of a cache of its own
            self.prefix = KvCache(be, 2, kv_heads, head_dim, prefix + 3, *types)
            pk, pv = fill(self.prefix, 2, prefix + 3)
            self.pk, self.pv = pk[1, :prefix], pv[1, :prefix]

    def run(self, heads, tokens, starts, counts=None, slots=None, window=0, scale=0.0, q=None):
        be, n = self.be, len(starts)
        slots = list(range(n)) if slots is None else slots
        shape = (n, tokens, heads, self.head_dim)
        self.q = q = self.rng.standard_normal(shape).astype(np.float32) if q is None else q
        out = DeviceArray.of(be, np.full(shape, SENTINEL, np.float32))
        ws = self.cache.attention_workspace(heads, n, tokens, self.prefix is not None)
        batch = self.cache.batch(tokens, _i32(be, slots), _i32(be, starts),
                                 None if counts is None else _i32(be, counts))
        self.cache.attention(DeviceArray.of(be, q), out, batch, workspace=ws, prefix=self.prefix,
                             prefix_slot=1 if self.prefix else 0, prefix_len=self.prefix_len, window=window, scale=scale)
        return out.get()

    def check(self, heads, tokens, starts, counts=None, slots=None, window=0, scale=0.0, q=None):
        got = self.run(heads, tokens, starts, counts, slots, window, scale, q)
        q, slots = self.q, list(range(len(starts))) if slots is None else slots
        for b, start in enumerate(starts):
            count = tokens if counts is None else max(0, min(tokens, counts[b]))
            low = max(0, -start)
            high = min(count, self.cache.capacity - start) if 0 <= slots[b] < self.cache.slots else 0
            inside = np.zeros(tokens, bool)
            if low < high:
                inside[low:high] = True
                k, v = self.k[slots[b], :start + high], self.v[slots[b], :start + high]
                if self.prefix is not None:
                    k, v = np.concatenate([self.pk, k]), np.concatenate([self.pv, v])
                want, tol = attend(q[b, low:high], k, v, self.prefix_len + start + low, window, scale or None)
                off = np.abs(got[b, low:high] - want)
                assert (off <= tol).all(), (b, float((off / tol).max()))
            assert (got[b, ~inside] == SENTINEL).all()
        return got


SHAPES = [(64, 1, 1), (64, 2, 4), (96, 3, 1), (128, 2, 4), (128, 1, 7), (256, 1, 2), (64, 1, 32)]


@pytest.mark.parametrize("head_dim,kv_heads,group", SHAPES)
@pytest.mark.parametrize("types", list(itertools.product((Q8_0, Q4_0), repeat=2)))
def test_single_tokens(hip, head_dim, kv_heads, group, types):
    """Sequences from one position to some hundreds, one token each."""
    lengths = [1, 2, 16, 31, 32, 33, 64, 100, 257, 700]
    case = Case(hip, kv_heads, head_dim, lengths, types, capacity=701, seed=head_dim + group)
    case.check(kv_heads * group, 1, [n - 1 for n in lengths])


@pytest.mark.parametrize("head_dim,kv_heads,group", SHAPES)
def test_several_tokens(hip, head_dim, kv_heads, group):
    """Drafted tokens: ragged counts, an empty sequence, a repeated slot, slots and positions that are not there."""
    lengths = [40, 95, 129, 300, 12]
    case = Case(hip, kv_heads, head_dim, lengths, capacity=300, seed=group)
    starts, counts = [35, 90, 120, 296, 6, 0, 10, -2, 298, 2 ** 31 - 1], [5, 3, 0, 4, 6, 1, 9, 6, 6, 6]
    case.check(kv_heads * group, 6, starts, counts, slots=[0, 1, 2, 3, 4, 1, 9, 0, 2, 0])


@pytest.mark.parametrize("tokens", [1, 3, 17, 70, 200])
@pytest.mark.parametrize("head_dim,kv_heads,group", [(64, 2, 4), (96, 2, 1), (128, 1, 8), (256, 1, 3)])
def test_prompts(hip, head_dim, kv_heads, group, tokens):
    """Prompts from an empty cache and behind a history, two at once."""
    case = Case(hip, kv_heads, head_dim, [tokens, tokens + 61], seed=tokens)
    case.check(kv_heads * group, tokens, [0, 61])


@pytest.mark.parametrize("head_dim,kv_heads,group,types", [(64, 8, 8, (Q8_0, Q4_0)), (96, 32, 1, (Q4_0, Q8_0)),
                                                           (128, 8, 4, (Q8_0, Q8_0)), (128, 8, 5, (Q4_0, Q4_0)),
                                                           (256, 4, 2, (Q8_0, Q8_0))])
def test_prompts_that_fill_the_card(hip, head_dim, kv_heads, group, types):
    """So many rows that tiles of 128 go in pairs (not at head_dim 256): an odd number of tiles, ragged prompts, one
    empty, some behind a history, a window."""
    tokens = 256 * 3 // group + 11
    batch = -(-256 // (kv_heads * 4)) + 1
    lengths = [tokens + 17 * b for b in range(batch)]
    starts = [17 * b for b in range(batch)]
    counts = [max(0, tokens - 60 * b) for b in range(batch)]
    if batch > 2:
        counts[2] = 0
    counts[1] = 1
    case = Case(hip, kv_heads, head_dim, lengths, types, seed=head_dim + group)
    case.check(kv_heads * group, tokens, starts, counts)
    case.check(kv_heads * group, tokens, starts, counts, window=45)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 250, 5000])
@pytest.mark.parametrize("prefix", [0, 150])
def test_window(hip, window, prefix):
    case = Case(hip, 2, 64, [300, 70, 1], prefix=prefix, capacity=300, seed=window)
    case.check(8, 4, [296, 66, 0], [4, 4, 1], window=window)
    case.check(8, 65, [230, 4, 0], [65, 65, 1], window=window)


@pytest.mark.parametrize("prefix", [1, 31, 32, 33, 500])
@pytest.mark.parametrize("head_dim,kv_heads,group", [(64, 2, 4), (96, 1, 1), (128, 2, 4), (256, 1, 2)])
def test_shared_prefix(hip, head_dim, kv_heads, group, prefix):
    lengths = [1, 40, 7, 33, 2, 90, 64, 5, 1, 17, 32]
    case = Case(hip, kv_heads, head_dim, lengths, prefix=prefix, capacity=90, seed=prefix)
    case.check(kv_heads * group, 1, [n - 1 for n in lengths])
    case.check(kv_heads * group, 3, [max(0, n - 3) for n in lengths], [min(3, n) for n in lengths])


def test_prefix_of_the_same_cache(hip):
    case = Case(hip, 2, 128, [20, 400, 35], seed=9)
    q = case.rng.standard_normal((2, 1, 8, 128)).astype(np.float32)
    out = DeviceArray(hip, q.shape)
    ws = case.cache.attention_workspace(8, 2, 1, True)
    case.cache.attention(DeviceArray.of(hip, q), out, case.cache.batch(1, _i32(hip, [0, 2]), _i32(hip, [19, 34])),
                         workspace=ws, prefix=case.cache, prefix_slot=1, prefix_len=333)
    got = out.get()
    for b, (slot, n) in enumerate([(0, 20), (2, 35)]):
        k = np.concatenate([case.k[1, :333], case.k[slot, :n]])
        v = np.concatenate([case.v[1, :333], case.v[slot, :n]])
        want, tol = attend(q[b], k, v, 333 + n - 1)
        assert (np.abs(got[b] - want) <= tol).all()


@pytest.mark.parametrize("types", [(Q8_0, Q8_0), (Q4_0, Q4_0)])
@pytest.mark.parametrize("what", ["large_v", "small_v", "mixed_v", "zero_v", "large_k", "flat", "sharp"])
def test_ranges(hip, types, what):
    """Values at the ends of the formats' range, rows whose scales differ by orders of magnitude, scores far apart."""
    def scaled(low, high):
        def change(x):
            p = np.random.default_rng(1).uniform(low, high, size=x.shape[:2] + (1, 1))
            return x * 10.0 ** p
        return change
    zero = np.arange(300) % 3 == 0

    def some_zero(x):
        x = x.copy()
        x[:, zero[:x.shape[1]]] = 0
        return x
    k_of = {"large_k": scaled(0, 2), "flat": lambda x: x * 1e-4, "sharp": lambda x: x * 30}.get(what)
    v_of = {"large_v": lambda x: x * 2e5, "small_v": lambda x: x * 1e-5, "mixed_v": scaled(-5, 5),
            "zero_v": some_zero}.get(what)
    case = Case(hip, 2, 128, [300, 45], types, k_of=k_of, v_of=v_of, seed=2)
    case.check(8, 1, [299, 44])
    case.check(8, 40, [255, 5])


def test_hidden_positions_do_not_reach_a_result(hip):
    """Rows behind a token's position and before its window: NaN, infinities and the largest values."""
    cases = []
    for bad in (None, np.nan, np.inf, -np.inf, 3e38):
        case = Case(hip, 1, 64, [128], seed=4)
        q = np.random.default_rng(8).standard_normal((1, 2, 4, 64)).astype(np.float32)
        if bad is not None:
            rows = np.full((1, 60, 1, 64), bad, np.float32)
            zero = _i32(hip, [0])
            for start, n in ((0, 20), (72, 56)):
                x = DeviceArray.of(hip, rows[:, :n])
                case.cache.write(x, x, case.cache.batch(n, zero, _i32(hip, [start])))
        cases.append(case.run(4, 2, [70], window=50, q=q))
    for got in cases[1:]:
        assert np.array_equal(got, cases[0])


def test_a_bad_query_row_stays_alone(hip):
    case = Case(hip, 1, 128, [200], seed=6)
    q = case.rng.standard_normal((1, 3, 4, 128)).astype(np.float32)
    want = case.run(4, 3, [190], q=q)
    for bad in (np.nan, np.inf, -np.inf):
        p = q.copy()
        p[0, 1, 2, 17] = bad
        got = case.run(4, 3, [190], q=p)
        keep = np.ones((3, 4), bool)
        keep[1, 2] = False
        assert np.array_equal(got[0][keep], want[0][keep])
        assert not np.isfinite(got[0, 1, 2]).all()


def test_scale(hip):
    case = Case(hip, 2, 64, [100, 33], seed=7)
    case.check(4, 2, [98, 31], scale=0.3)
    case.check(4, 2, [98, 31], scale=1e-20)


def test_positions_past_four_gigabytes(hip):
    cap = 1 << 20
    rng = np.random.default_rng(12)
    with KvCache(hip, 5, 8, 128, cap) as cache:
        k = rng.standard_normal((1, 100, 8, 128)).astype(np.float32)
        v = rng.standard_normal((1, 100, 8, 128)).astype(np.float32)
        slot = _i32(hip, [4])
        cache.write(DeviceArray.of(hip, k), DeviceArray.of(hip, v), cache.batch(100, slot, _i32(hip, [cap - 100])))
        q = rng.standard_normal((1, 2, 8, 128)).astype(np.float32)
        out = DeviceArray(hip, q.shape)
        cache.attention(DeviceArray.of(hip, q), out, cache.batch(2, slot, _i32(hip, [cap - 2])),
                        workspace=cache.attention_workspace(8, 1, 2), window=90)
        want, tol = attend(q[0], held(k[0], Q8_0), held(v[0], Q8_0), 98, 90)
        assert (np.abs(out.get()[0] - want) <= tol).all()


def test_same_bits_every_time(hip):
    """Splits of the keys are summed in one order: repeated calls agree bit for bit."""
    case = Case(hip, 2, 128, [3000, 1500, 9], capacity=3000, prefix=700, seed=3)
    q = case.rng.standard_normal((3, 1, 8, 128)).astype(np.float32)
    first = case.run(8, 1, [2999, 1499, 8], q=q)
    for _ in range(3):
        assert np.array_equal(case.run(8, 1, [2999, 1499, 8], q=q), first)
    case.check(8, 1, [2999, 1499, 8], q=q)


def test_refusals(hip):
    cache = KvCache(hip, 2, 2, 64, 64)
    other = KvCache(hip, 1, 2, 64, 64, k_type=Q4_0)
    one = _i32(hip, [0])
    batch = cache.batch(1, one, one)
    q, out = DeviceArray(hip, (1, 1, 4, 64)), DeviceArray(hip, (1, 1, 4, 64))
    ws = cache.attention_workspace(4, 1, 1, True)
    cache.attention(q, out, batch, workspace=ws, prefix=cache, prefix_len=64)
    odd = DeviceArray(hip, (1, 1, 3, 64))
    for kwargs, exc in [(dict(window=-1), ValueError), (dict(scale=-1.0), ValueError), (dict(scale=float("nan")), ValueError),
                        (dict(prefix_len=3), ValueError), (dict(prefix=cache, prefix_len=-1), ValueError),
                        (dict(prefix=cache, prefix_len=65), IndexError),
                        (dict(prefix=cache, prefix_slot=2, prefix_len=4), IndexError),
                        (dict(prefix=other, prefix_len=4), ValueError)]:
        with pytest.raises(exc):
            cache.attention(q, out, batch, workspace=ws, **kwargs)
    with pytest.raises(ValueError):
        cache.attention(odd, odd, batch, workspace=ws)
    with pytest.raises(ValueError):
        cache.attention(q, odd, batch, workspace=ws)
    with pytest.raises(ValueError):
        cache.attention_workspace(3, 1, 1)
    with pytest.raises(ValueError):
        cache.attention_workspace(4, -1, 1)


@pytest.mark.parametrize("head_dim,kv_heads,group", [(64, 2, 4), (128, 1, 2), (256, 2, 7)])
@pytest.mark.parametrize("window", [1, 20, 32, 70])
def test_prompt_that_leaves_its_prefix_behind(hip, head_dim, kv_heads, group, window):
    """Windows that only the first rows of a prompt share with the prefix, in a workspace that holds NaN where parts
    are not written."""
    case = Case(hip, kv_heads, head_dim, [200, 131], prefix=90, capacity=200, seed=window)
    ws = case.cache.attention_workspace(kv_heads * group, 2, 131, True)
    fill = np.zeros(ws.nbytes, np.uint8)
    fill[1 << 19:] = 255          # behind the counters
    ws.put(fill)
    case.cache.attention_workspace = lambda *a: ws
    case.check(kv_heads * group, 131, [69, 0], [131, 100], window=window)
    case.check(kv_heads * group, 131, [0, 0], [5, 131], window=window)


def test_workspace_with_a_prefix_serves_calls_without(hip):
    """Whatever the plan: the larger of the two."""
    cache = KvCache(hip, 1, 1, 64, 4000)
    for heads in (1, 2, 8):
        for batch, tokens in ((1, 1), (1, 500), (1, 2065), (3, 700), (129, 1), (300, 5), (500, 1)):
            assert (cache.attention_workspace(heads, batch, tokens, True).nbytes
                    >= cache.attention_workspace(heads, batch, tokens).nbytes)
