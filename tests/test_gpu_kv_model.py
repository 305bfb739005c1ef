"""InferenceEngine over a quantised KV cache, against a 64-bit NumPy forward whose
keys and values are rounded as the cache holds them."""
import numpy as np
import pytest

from dotllm_amd import Q4_0, Q8_0, InferenceEngine, LoadedModel, synth
from dotllm_amd.engine import greedy
from tests.kv_reference import held
from tests.test_oracle_forward import Forward

pytestmark = pytest.mark.gpu

TYPES = {"q8_0": Q8_0, "q4_0": Q4_0}


class _Held:
    """K or V rows [layers, context, kv_heads, head_dim] that are rounded as they are stored."""

    def __init__(self, rows, kind):
        self.rows, self.kind = rows, kind

    def __setitem__(self, at, x):
        self.rows[at] = held(np.asarray(x, dtype=np.float32), self.kind)

    def __getitem__(self, at):
        return self.rows[at]


class HeldForward(Forward):
    def __init__(self, img, context, kind):
        super().__init__(img, context)
        self.K, self.V = _Held(self.K, kind), _Held(self.V, kind)

    def softmax(self, s):   # the exact exponential
        e = np.exp(s - s.max())
        return e / e.sum()


# A key or value next to a border between two integers may round the other way than in 64 bits: one step of its
# block, 1/127 (Q8_0) or 1/8 (Q4_0) of the block's largest, in one of head_dim elements of one position.  Everything
# else is 32-bit arithmetic, whose share the tests of the fp32 cache bound by 2e-2; the bound of those tests is kept.
TOL = 2e-2


@pytest.mark.parametrize("kv_type", ["q8_0", "q4_0"])
@pytest.mark.parametrize("name,extra", [("tiny", {}), ("tiny", dict(sliding_window=9)),
                                        ("small5", dict(fused_qkv=True, qk_norm=True))])
def test_logits(hip, kv_type, name, extra):
    img = synth.build_image(name, seed=21, context=64, **extra)
    tokens = synth.prompt(32000, 45, seed=5)
    ref = HeldForward(img, 64, TYPES[kv_type])
    want = [ref.step(int(t), p) for p, t in enumerate(tokens)]
    with InferenceEngine(LoadedModel.load(img), hip, kv_type=kv_type) as eng:
        # a prompt as one chunk, then single tokens; then all of it token by token; then two chunks
        logits, _ = eng.prefill(tokens[:40])
        assert np.max(np.abs(logits - want[39])) <= TOL
        for p in range(40, 45):
            assert np.max(np.abs(eng.process_token(int(tokens[p]), p) - want[p])) <= TOL
        for layer in (0, ref.cfg.layer_count - 1):
            k, v = eng.kv_read(layer, 41)
            # a row's own rounding: a step of its largest block at most
            step = 1 / 127 if kv_type == "q8_0" else 1 / 8
            for got, rows in ((k, ref.K), (v, ref.V)):
                w = rows[layer, 41].reshape(-1)
                assert np.max(np.abs(got - w)) <= 1.1 * step * np.abs(w).max()
        eng.reset()
        for p in range(45):
            got = eng.process_token(int(tokens[p]), p)
        assert np.max(np.abs(got - want[44])) <= TOL
        eng.prefill(tokens[:17])
        logits, _ = eng.prefill(tokens[17:45], 17)
        assert np.max(np.abs(logits - want[44])) <= TOL


def test_generate(hip, tiny_image):
    """Greedy generation through the captured step: the same tokens as single steps give, and again after a reset."""
    prompt = synth.prompt(32000, 20, seed=3)
    with InferenceEngine(LoadedModel.load(tiny_image), hip, kv_type="q8_0") as eng:
        tokens, logits = eng.generate_all(prompt, greedy(40), return_logits=True)
        assert eng.generate_all(prompt, greedy(40))[0] == tokens
        assert list(eng.generate(prompt, greedy(40), chunk=7)) == tokens
        one, _ = eng.prefill(prompt)
        assert np.array_equal(one, logits[0])
        for i, t in enumerate(tokens[:5]):
            assert np.array_equal(eng.process_token(t, 20 + i), logits[i + 1])
        assert eng.step_bytes(100) < 1e9
        with pytest.raises(NotImplementedError):
            eng.kv_fill_random(8)


def test_refused_type(hip, tiny_image):
    with pytest.raises(ValueError):
        InferenceEngine(LoadedModel.load(tiny_image), hip, kv_type="q5_0")
