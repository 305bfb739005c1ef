"""HipBackend.verify_drafts against a plain 64-bit form: the same tokens."""
import numpy as np
import pytest

from dotllm_amd import DeviceArray
from tests.kv_reference import verify

pytestmark = pytest.mark.gpu


def run(be, target, drafts, uniforms, temperature, draft=None, counts=None):
    b, n1, vocab = target.shape
    tokens = DeviceArray.of(be, np.full((b, n1), -9, np.int32))
    accepted = DeviceArray.of(be, np.full(b, -9, np.int32))
    be.verify_drafts(DeviceArray.of(be, target, np.float32), DeviceArray.of(be, drafts, np.int32),
                     DeviceArray.of(be, uniforms, np.float32), tokens, accepted, temperature=temperature,
                     workspace=be.verify_workspace(b, n1 - 1, vocab),
                     draft=None if draft is None else DeviceArray.of(be, draft, np.float32),
                     counts=None if counts is None else DeviceArray.of(be, counts, np.int32))
    return tokens.get(), accepted.get()


def check(be, target, drafts, uniforms, temperature, draft=None, counts=None):
    tokens, accepted = run(be, target, drafts, uniforms, temperature, draft, counts)
    for b in range(target.shape[0]):
        want, a = verify(target[b], drafts[b], uniforms[b], temperature, None if draft is None else draft[b],
                         None if counts is None else counts[b])
        assert accepted[b] == a and np.array_equal(tokens[b], want), (b, tokens[b], want)
    return accepted


def logits(rng, b, n, vocab):
    """Target and draft logits that mostly agree, and drafts drawn from the draft's."""
    target = rng.standard_normal((b, n + 1, vocab)).astype(np.float32) * 2
    draft = (target[:, :n] + rng.standard_normal((b, n, vocab)) * 0.6).astype(np.float32)
    e = np.exp(draft.astype(np.float64) / 0.8)
    cum = (e / e.sum(-1, keepdims=True)).cumsum(-1)
    drafts = (cum <= rng.random((b, n, 1))).sum(-1).clip(max=vocab - 1).astype(np.int32)
    return target, draft, drafts, rng.random((b, n + 1), dtype=np.float32)


@pytest.mark.parametrize("vocab", [1, 2, 63, 257, 1000, 4099, 32000])
@pytest.mark.parametrize("with_draft", [True, False])
def test_sampled(hip, vocab, with_draft):
    rng = np.random.default_rng(vocab)
    target, draft, drafts, u = logits(rng, 6, 5, vocab)
    for t in (0.8, 1.0, 0.3):
        check(hip, target, drafts, u, t, draft if with_draft else None)
        check(hip, target, drafts, u, t, draft if with_draft else None, [5, 0, 1, 3, -2, 99])


def test_every_number_of_accepted_drafts_occurs(hip):
    rng = np.random.default_rng(4)
    target, draft, drafts, u = logits(rng, 64, 3, 500)
    seen = set(check(hip, target, drafts, u, 0.8, draft).tolist())
    assert seen == {0, 1, 2, 3}


@pytest.mark.parametrize("drafts_n", [0, 1, 8, 40])
def test_number_of_drafts(hip, drafts_n):
    rng = np.random.default_rng(drafts_n)
    target, draft, drafts, u = logits(rng, 3, drafts_n, 700)
    u[:, :-1] *= 0.3
    check(hip, target, drafts, u, 0.9, draft)
    check(hip, target, drafts, u, 0.9)


def test_greedy(hip):
    rng = np.random.default_rng(7)
    target, _, drafts, u = logits(rng, 9, 4, 3001)
    best = target.argmax(-1).astype(np.int32)
    drafts = best[:, :4].copy()
    drafts[1, 0] += 1
    drafts[2, 2] = 0
    drafts[3, 3] = -1
    target[4, 1, 5] = target[4, 1, 2999] = 50.0   # the first of equal maxima
    drafts[4, 1] = 2999
    target[5, 0, :] = np.nan                        # a row without a maximum
    target[6, 0, 0] = np.nan
    target[7, 2, :] = -np.inf
    for t in (0.0, -1.0):
        check(hip, target, drafts, u, t)
        check(hip, target, drafts, u, t, counts=[4, 4, 1, 4, 4, 4, 0, 4, 2])


def test_masked_and_infinite_logits(hip):
    """-infinity (a token that must not come), NaN, +infinity, rows without mass, ids outside the vocabulary."""
    rng = np.random.default_rng(9)
    target, draft, drafts, u = logits(rng, 10, 3, 600)
    target[0, :, ::2] = -np.inf
    draft[1, :, 1::2] = -np.inf
    target[2, 1, :] = -np.inf
    target[3, 0, 17] = np.inf
    target[3, 1, [5, 80]] = np.inf
    draft[4, 0, :] = np.nan
    target[5, :, 100:200] = np.nan
    drafts[6, 0], drafts[7, 1], drafts[8, 2] = -1, 600, 2 ** 31 - 1
    draft[9, 0, drafts[9, 0]] = np.inf
    for t in (0.8, 2.0):
        check(hip, target, drafts, u, t, draft)
        check(hip, target, drafts, u, t)


def test_draws_at_the_ends(hip):
    """Draws of 0 and of the largest number below 1; the same rows for target and draft (nothing is ever left over)."""
    rng = np.random.default_rng(2)
    target, draft, drafts, u = logits(rng, 4, 3, 900)
    for value in (0.0, float(np.nextafter(np.float32(1), np.float32(0)))):
        u[:] = value
        check(hip, target, drafts, u, 0.8, draft)
        check(hip, target, drafts, u, 0.8)
        assert (check(hip, target, drafts, u, 0.8, target[:, :3].copy()) == 3).all()


def test_rows_may_start_anywhere(hip):
    """Odd vocabularies: rows that begin at every alignment of 4 bytes."""
    rng = np.random.default_rng(6)
    for vocab in (5, 1001, 1002, 1003, 2047):
        target, draft, drafts, u = logits(rng, 3, 3, vocab)
        check(hip, target, drafts, u, 0.7, draft)


def test_accepted_tokens_follow_the_target(hip):
    """Over many draws the first token is distributed as the target alone: sqrt(p (1 - p) / n) is the deviation of
    each frequency; 5 of them for 8 tokens leave a chance below 1e-5."""
    rng = np.random.default_rng(1)
    b, vocab = 4096, 8
    target = np.broadcast_to(rng.standard_normal((1, 2, vocab)), (b, 2, vocab)).astype(np.float32)
    draft = np.broadcast_to(rng.standard_normal((1, 1, vocab)), (b, 1, vocab)).astype(np.float32)
    q = np.exp(draft[0, 0].astype(np.float64))
    drafts = rng.choice(vocab, size=(b, 1), p=q / q.sum()).astype(np.int32)
    tokens, _ = run(hip, target, drafts, rng.random((b, 2), dtype=np.float32), 1.0, draft)
    p = np.exp(target[0, 0].astype(np.float64))
    p /= p.sum()
    got = np.bincount(tokens[:, 0], minlength=vocab) / b
    assert (np.abs(got - p) <= 5 * np.sqrt(p * (1 - p) / b)).all()


def test_refusals(hip):
    f = lambda *s: DeviceArray(hip, s)                      # noqa: E731
    i = lambda *s: DeviceArray(hip, s, "int32")             # noqa: E731
    ws = hip.verify_workspace(2, 3, 50)
    ok = dict(temperature=1.0, workspace=ws)
    hip.verify_drafts(f(2, 4, 50), i(2, 3), f(2, 4), i(2, 4), i(2), **ok)
    for args in [(f(2, 4, 50), i(2, 4), f(2, 4), i(2, 4), i(2)), (f(2, 4, 50), f(2, 3), f(2, 4), i(2, 4), i(2)),
                 (f(2, 4, 50), i(2, 3), f(2, 3), i(2, 4), i(2)), (f(2, 4, 50), i(2, 3), f(2, 4), i(2, 3), i(2)),
                 (f(2, 4, 50), i(2, 3), f(2, 4), i(2, 4), i(3)), (np.zeros((2, 4, 50)), i(2, 3), f(2, 4), i(2, 4), i(2))]:
        with pytest.raises(ValueError):
            hip.verify_drafts(*args, **ok)
    with pytest.raises(ValueError):
        hip.verify_drafts(f(2, 4, 50), i(2, 3), f(2, 4), i(2, 4), i(2), temperature=float("nan"), workspace=ws)
    with pytest.raises(ValueError):
        hip.verify_drafts(f(2, 4, 50), i(2, 3), f(2, 4), i(2, 4), i(2), draft=f(2, 4, 50), **ok)
    with pytest.raises(NotImplementedError):
        hip.verify_workspace(1, 1, (1 << 24) + 1)
    with pytest.raises(ValueError):
        hip.verify_workspace(1, -1, 100)


@pytest.mark.parametrize("size", [1.0, 1e12, 1e30, 3e38])
@pytest.mark.parametrize("temperature", [1e-30, 0.8, 1e20, 3e38])
def test_far_apart(hip, size, temperature):
    """Logits between which floats lie further apart than any mass reaches, temperatures at the ends of their range,
    logits without mass among them."""
    rng = np.random.default_rng(17)
    target, draft, drafts, u = logits(rng, 4, 3, 1500)
    for x in (target, draft):
        x[:] = (x / np.abs(x).max() * size).astype(np.float32)
        x[0, :, ::3] = -np.inf
        x[1, :, ::2] = np.nan
        x[2, :, :1499] = -np.inf
    drafts[0] = target[0, :3].argmax(-1)
    drafts[2] = 1499
    check(hip, target, drafts, u, temperature, draft)
    check(hip, target, drafts, u, temperature)
