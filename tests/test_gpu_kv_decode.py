"""The cache's operators as a serving loop calls them: one after the other, with one
workspace, eagerly and as a captured graph."""
import ctypes as C

import numpy as np
import pytest

from dotllm_amd import Q4_0, Q8_0, DeviceArray, KvCache, _lib
from tests.kv_reference import attend, held, verify

pytestmark = pytest.mark.gpu

HEADS, KV, HD, VOCAB = 6, 2, 64, 1500


class Loop:
    """Decoding with drafted tokens: three sequences behind a shared prefix, ragged prompts, `drafts` drafted tokens a
    round, of which some sequences use fewer."""

    def __init__(self, be, types, drafts, seed):
        rng = self.rng = np.random.default_rng(seed)
        self.be, self.drafts, self.types = be, drafts, types
        self.embed = [rng.standard_normal((VOCAB, h, HD)).astype(np.float32) for h in (HEADS, KV, KV)]
        self.cache = KvCache(be, 5, KV, HD, 200, *types)
        self.slots, self.prompts = [4, 1, 2], [rng.integers(VOCAB, size=n) for n in (17, 1, 40)]
        self.prefix = rng.integers(VOCAB, size=35)
        self.past = [list(p) for p in self.prompts]     # tokens whose rows are in the cache
        b, n = 3, drafts + 1
        arr = lambda shape, t=np.float32: DeviceArray(be, shape, t)
        self.q, self.out, self.k, self.v = arr((b, n, HEADS, HD)), arr((b, n, HEADS, HD)), arr((b, n, KV, HD)), arr((b, n, KV, HD))
        self.starts, self.counts, self.used = arr(b, np.int32), arr(b, np.int32), arr(b, np.int32)
        self.batch = self.cache.batch(n, DeviceArray.of(be, self.slots, np.int32), self.starts, self.counts)
        self.target, self.draft_ids = arr((b, n, VOCAB)), arr((b, drafts), np.int32)
        self.uniforms, self.tokens, self.accepted = arr((b, n)), arr((b, n), np.int32), arr(b, np.int32)
        sizes = [self.cache.attention_workspace(HEADS, b, n, True), be.verify_workspace(b, drafts, VOCAB)]
        self.work = max(sizes, key=lambda w: w.nbytes)
        # the prefix in slot 0, then the prompts as one padded batch
        self.fill([0], [self.prefix])
        self.fill(self.slots, self.prompts)
        self.cur = rng.integers(VOCAB, size=b)
        self.round = 0

    def fill(self, slots, prompts):
        n = max(len(p) for p in prompts)
        ids = np.stack([np.pad(p, (0, n - len(p))) for p in prompts])
        i32 = lambda v: DeviceArray.of(self.be, v, np.int32)
        self.cache.write(DeviceArray.of(self.be, self.embed[1][ids]), DeviceArray.of(self.be, self.embed[2][ids]),
                         self.cache.batch(n, i32(slots), i32(np.zeros(len(slots))), i32([len(p) for p in prompts])))

    def put(self):
        """A round's inputs; the target's logits favour most of the drafts."""
        rng, n = self.rng, self.drafts
        self.n = np.array([n, max(0, n - 1), (self.round * 2) % (n + 1)])
        self.d = rng.integers(VOCAB, size=(3, n)).astype(np.int32)
        ids = self.ids = np.concatenate([self.cur[:, None], self.d], 1)
        logits = rng.standard_normal((3, n + 1, VOCAB)).astype(np.float32)
        keep = rng.random((3, n)) < 0.7
        np.put_along_axis(logits[:, :n], self.d[:, :, None], np.where(keep, 9.0, -2.0)[:, :, None].astype(np.float32), 2)
        self.logits, self.u = logits, rng.random((3, n + 1), dtype=np.float32)
        for a, x in [(self.q, self.embed[0][ids]), (self.k, self.embed[1][ids]), (self.v, self.embed[2][ids]),
                     (self.starts, [len(p) for p in self.past]), (self.counts, self.n + 1), (self.used, self.n),
                     (self.target, logits), (self.draft_ids, self.d), (self.uniforms, self.u),
                     (self.out, np.zeros(self.out.shape)), (self.tokens, np.full((3, n + 1), -9)),
                     (self.accepted, np.full(3, -9))]:
            a.put(x)

    def run(self):
        self.cache.write(self.k, self.v, self.batch)
        self.cache.attention(self.q, self.out, self.batch, workspace=self.work, prefix=self.cache, prefix_slot=0,
                             prefix_len=len(self.prefix), window=60)
        self.be.verify_drafts(self.target, self.draft_ids, self.uniforms, self.tokens, self.accepted, temperature=0.7,
                              workspace=self.work, counts=self.used)

    def check(self):
        out, tokens, accepted = self.out.get(), self.tokens.get(), self.accepted.get()
        for b in range(3):
            n = int(self.n[b]) + 1
            ids = np.concatenate([self.prefix, self.past[b], self.ids[b, :n]])
            want, tol = attend(self.embed[0][self.ids[b, :n]], held(self.embed[1][ids], self.types[0]),
                               held(self.embed[2][ids], self.types[1]), len(ids) - n, 60)
            assert (np.abs(out[b, :n] - want) <= tol).all()
            assert (out[b, n:] == 0).all()
            wt, wa = verify(self.logits[b], self.d[b], self.u[b], 0.7, count=self.n[b])
            assert accepted[b] == wa and np.array_equal(tokens[b], wt)
            # the standing tokens stay; rejected drafts' rows are written over in the next round
            self.past[b] += list(self.ids[b, :wa + 1])
            self.cur[b] = tokens[b, wa]
        self.round += 1
        return accepted


@pytest.mark.parametrize("drafts", [0, 1, 4])
@pytest.mark.parametrize("types", [(Q8_0, Q8_0), (Q8_0, Q4_0)])
def test_loop(hip, drafts, types):
    loop = Loop(hip, types, drafts, seed=drafts)
    stood = []
    for _ in range(8):
        loop.put()
        loop.run()
        stood += loop.check().tolist()
    if drafts == 4:
        assert len(set(stood)) >= 3


class Graphs:
    """Capture on a backend's stream, through the HIP runtime that its library has loaded."""

    def __init__(self, be):
        with open("/proc/self/maps") as f:
            path = next(line.split()[-1] for line in f if "libamdhip64" in line)
        self.hip, self.stream, self.be = C.CDLL(path), C.c_void_p(be.stream), be

    def call(self, name, *args):
        assert getattr(self.hip, name)(*args) == 0, name

    def capture(self, run):
        self.be.synchronize()
        graph, runner = C.c_void_p(), C.c_void_p()
        self.call("hipStreamBeginCapture", self.stream, C.c_int(0))
        run()
        self.call("hipStreamEndCapture", self.stream, C.byref(graph))
        self.call("hipGraphInstantiate", C.byref(runner), graph, None, None, C.c_size_t(0))
        self.call("hipGraphDestroy", graph)
        return runner

    def launch(self, runner):
        self.call("hipGraphLaunch", runner, self.stream)

    def free(self, runner):
        self.be.synchronize()
        self.call("hipGraphExecDestroy", runner)


@pytest.mark.parametrize("drafts", [0, 4])
def test_captured_loop(hip, drafts):
    """The loop's step as a graph, replayed with new positions, counts and contents; eager calls of other sizes use the
    workspace in between, and an eager loop gives the same bits."""
    loop, eager = (Loop(hip, (Q8_0, Q8_0), drafts, seed=11) for _ in range(2))
    graphs = Graphs(hip)
    runner = graphs.capture(loop.run)
    two = graphs.capture(loop.run)          # a second graph that shares the workspace
    rng = np.random.default_rng(2)
    for i in range(6):
        loop.put()
        graphs.launch(two if i % 3 == 2 else runner)
        eager.put()
        eager.run()
        for a, b in ((loop.out, eager.out), (loop.tokens, eager.tokens), (loop.accepted, eager.accepted)):
            assert np.array_equal(a.get(), b.get())
        loop.check()
        eager.check()
        # something else in the same workspace
        n = [1, 9, 30][i % 3]
        q = rng.standard_normal((1, n, HEADS, HD)).astype(np.float32)
        work = max(loop.work, hip.verify_workspace(1, 0, VOCAB), loop.cache.attention_workspace(HEADS, 1, n),
                   key=lambda w: w.nbytes)
        out = DeviceArray(hip, q.shape)
        i32 = lambda v: DeviceArray.of(hip, v, np.int32)
        loop.cache.attention(DeviceArray.of(hip, q), out, loop.cache.batch(n, i32([0]), i32([35 - n])), workspace=work)
        want, tol = attend(q[0], held(loop.embed[1][loop.prefix], Q8_0), held(loop.embed[2][loop.prefix], Q8_0), 35 - n)
        assert (np.abs(out.get()[0] - want) <= tol).all()
    graphs.free(runner)
    graphs.free(two)


def test_one_workspace_for_all(hip):
    """Attention in chunks (whose counters and parts fill the workspace), drafts of many sequences, back and forth."""
    rng = np.random.default_rng(5)
    cache = KvCache(hip, 3, 4, 64, 2000)
    x = [rng.standard_normal((3, 2000, 4, 64)).astype(np.float32) for _ in range(2)]
    i32 = lambda v: DeviceArray.of(hip, v, np.int32)
    cache.write(*(DeviceArray.of(hip, a) for a in x), cache.batch(2000, i32([0, 1, 2]), i32([0, 0, 0])))
    hk, hv = held(x[0], Q8_0), held(x[1], Q8_0)
    b, vocab = 600, 1100
    target = rng.standard_normal((b, 2, vocab)).astype(np.float32)
    drafts, u = rng.integers(vocab, size=(b, 1)).astype(np.int32), rng.random((b, 2), dtype=np.float32)
    dev = [DeviceArray.of(hip, a) for a in (target, drafts, u)]
    need = max(hip.verify_workspace(b, 1, vocab).nbytes, cache.attention_workspace(16, 3, 3, True).nbytes,
               cache.attention_workspace(16, 3, 40).nbytes)
    work = DeviceArray(hip, (need,), "uint8")
    for step in range(4):
        for n, prefix in ((1, 0), (3, 0), (40, 0), (1, 500)):
            q = rng.standard_normal((3, n, 16, 64)).astype(np.float32)
            out, starts = DeviceArray(hip, q.shape), [1999 - n, 700, 1500]
            cache.attention(DeviceArray.of(hip, q), out, cache.batch(n, i32([0, 1, 2]), i32(starts)), workspace=work,
                            prefix=cache if prefix else None, prefix_slot=1, prefix_len=prefix)
            got = out.get()
            for s in range(3):
                k, v = hk[s, :starts[s] + n], hv[s, :starts[s] + n]
                if prefix:
                    k, v = np.concatenate([hk[1, :prefix], k]), np.concatenate([hv[1, :prefix], v])
                want, tol = attend(q[s], k, v, len(k) - n)
                assert (np.abs(got[s] - want) <= tol).all()
            tokens, accepted = DeviceArray(hip, (b, 2), "int32"), DeviceArray.of(hip, np.full(b, -9, np.int32))
            hip.verify_drafts(*dev, tokens, accepted, temperature=1.0, workspace=work)
            got, stood = tokens.get(), accepted.get()
            if step == 0 and not prefix and n == 1:
                wants = [verify(target[i], drafts[i], u[i], 1.0) for i in range(b)]
            assert stood.tolist() == [w[1] for w in wants]
            assert np.array_equal(got, np.stack([w[0] for w in wants]))


def test_empty_calls(hip):
    """No sequences or no tokens: nothing to do, whatever the (empty) arrays' addresses."""
    cache = KvCache(hip, 1, 2, 64, 64)
    for b, t in ((0, 5), (5, 0), (0, 0)):
        rows = _lib.TokenBatch(b, t, None, None, None)
        opt = _lib.Attention(2, 0, 0.0, None, 0, 0, 0, 0)
        L = _lib.lib()
        _lib.call(L.llmdot_hip_kv_cache_write(cache.handle, None, 0, None, 0, C.byref(rows)))
        _lib.call(L.llmdot_hip_kv_cache_read(cache.handle, None, 0, None, 0, C.byref(rows)))
        _lib.call(L.llmdot_hip_kv_cache_attention(cache.handle, None, None, C.byref(rows), C.byref(opt), None, 0))
    empty = [DeviceArray(hip, s, t) for s, t in (((0, 4, 10), "float32"), ((0, 3), "int32"), ((0, 4), "float32"),
                                                 ((0, 4), "int32"), ((0,), "int32"))]
    hip.verify_drafts(*empty, temperature=1.0, workspace=hip.verify_workspace(0, 3, 10))


def test_refused_sizes(hip):
    cache = KvCache(hip, 1, 2, 64, 300)
    q, one = DeviceArray(hip, (1, 1, 4, 64)), DeviceArray(hip, (1,), "int32")
    small = DeviceArray(hip, (cache.attention_workspace(4, 1, 1).nbytes - 1,), "uint8")
    with pytest.raises(ValueError):
        cache.attention(q, q, cache.batch(1, one, one), workspace=small)
    many = DeviceArray(hip, (4097,), "int32")
    with pytest.raises(NotImplementedError):
        cache.attention_workspace(4, 4097, 1)
    with pytest.raises(NotImplementedError):
        cache.write(*(DeviceArray(hip, (4097, 1, 2, 64)),) * 2, cache.batch(1, many, many))
    target = DeviceArray(hip, (2, 1, 50))
    tokens, none = DeviceArray(hip, (2, 1), "int32"), DeviceArray(hip, (2, 0), "int32")
    with pytest.raises(ValueError):
        hip.verify_drafts(target, none, DeviceArray(hip, (2, 1)), tokens, DeviceArray(hip, (2,), "int32"),
                          temperature=1.0, workspace=DeviceArray(hip, (16,), "uint8"))
    for sizes in ((4097, 1, 50), (1, 1025, 50), (1, 1, (1 << 24) + 1)):
        with pytest.raises(NotImplementedError):
            hip.verify_workspace(*sizes)
