"""Plain 64-bit forms of the operators over device memory, and their test tolerances."""
import math

import numpy as np

from dotllm_amd import Q8_0, synth
from oracle import oracle as O

U = 2.0 ** -24   # half a step of fp32, relative


def held(x, ggml_type):
    """What a cache of that type holds for finite rows x [..., head_dim]: the package's host quantiser, decoded by the
    oracle.  Blocks whose scale passes fp16's largest (the quantiser then has no number for them) are held with the
    largest, as the cache documents."""
    flat = np.ascontiguousarray(x, dtype=np.float32).reshape(-1, x.shape[-1])
    if flat.shape[0] == 0:
        return flat.astype(np.float64).reshape(x.shape)
    y = O.dequantize(synth.quantize(ggml_type, flat), ggml_type, flat.shape[0], flat.shape[1])
    y = y.astype(np.float64).reshape(-1, 32)
    for block in np.nonzero(~np.isfinite(y).all(-1))[0]:
        v = flat.reshape(-1, 32)[block].astype(np.float64)
        low, high = (-127, 127) if ggml_type == Q8_0 else (-8, 7)
        scale = 65504.0 if ggml_type == Q8_0 else -65504.0 * np.sign(v[np.argmax(np.abs(v))])
        r = (v / scale).astype(np.float32).astype(np.float64)
        y[block] = np.clip(np.sign(r) * np.floor(np.abs(r) + 0.5), low, high) * scale
    return y.reshape(x.shape)


def attend(q, k, v, first, window=0, scale=None):
    """q [n, heads, hd] at positions first .. first + n - 1 over k, v [positions, kv_heads, hd] (positions 0 ..), and a
    bound on what 32-bit arithmetic of the documented kind may be off by, per element.

    A weight's relative error is its score's absolute error: the product's sums of hd terms in 32 bits and the query's
    22-bit significand, (hd + 16) U of sum |q k| scale, then a few roundings of the score itself and of exp2 (16 U and
    6 U |s|).  Weights enter the products with 22 bits (8 U) and sums over n positions round at most n times, in the
    numerator and the denominator: with |v| at most m, out is off by at most 2 m (weight error + 8 U + n U)."""
    n, heads, hd = q.shape
    group = heads // k.shape[1]
    scale = scale or 1.0 / math.sqrt(hd)
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    at, key = first + np.arange(n)[:, None], np.arange(k.shape[0])[None, :]
    seen = (key <= at) & (key > at - window) if window else key <= at
    count = seen.sum(-1)
    for h in range(heads):
        kk, vv, qq = k[:, h // group], v[:, h // group], q[:, h].astype(np.float64)
        s = np.where(seen, (qq @ kk.T) * scale, -np.inf)
        e = np.exp(s - s.max(-1, keepdims=True))
        out[:, h] = (e @ vv) / e.sum(-1, keepdims=True)
        mag = np.where(seen, np.abs(qq) @ np.abs(kk).T, 0.0).max(-1) * scale
        most = np.where(seen, np.abs(s), 0.0).max(-1)
        off = (hd + 16) * U * mag + 16 * U + 6 * U * most
        vmax = np.where(seen, np.abs(vv).max(-1)[None, :], 0.0).max(-1)
        tol[:, h] = (2 * vmax * (off + 8 * U + count * U))[:, None]
    return out, tol


def verify(target, drafts, uniforms, temperature, draft=None, count=None):
    """One sequence: target [n + 1, vocab], drafts [n], uniforms [n + 1]; (tokens [n + 1], accepted)."""
    n, vocab = drafts.shape[0], target.shape[1]
    count = n if count is None else max(0, min(n, count))

    def probs(x):
        x = x.astype(np.float64)
        x = np.where(np.isnan(x), -np.inf, x)
        top = x.max()
        if top == np.inf:
            e = (x == np.inf).astype(np.float64)
        elif top == -np.inf:
            return np.zeros(vocab)
        else:
            e = np.exp((x - top) / np.float64(np.float32(temperature)))
        return e / e.sum()

    def first_max(x):
        x = np.where(np.isnan(x), -np.inf, x)
        return int(np.argmax(x)) if x.max() > -np.inf else -1

    a = 0
    while a < count:
        t = int(drafts[a])
        if temperature <= 0:
            if first_max(target[a]) != t:
                break
        else:
            q = 1.0 if draft is None else (probs(draft[a])[t] if 0 <= t < vocab else 1.0)
            if not (0 <= t < vocab and float(uniforms[a]) * q < probs(target[a])[t]):
                break
        a += 1
    if temperature <= 0:
        nxt = first_max(target[a])
    else:
        p = probs(target[a])
        r = p
        if a < count:
            if draft is not None:
                q = probs(draft[a])
            else:
                q = np.zeros(vocab)
                if 0 <= drafts[a] < vocab:
                    q[drafts[a]] = 1.0
            r = np.maximum(p - q, 0.0)
            if not r.sum() > 0:
                r = p
        nxt = -1
        if r.sum() > 0:
            cum = np.cumsum(r)
            over = np.nonzero((cum > float(uniforms[n]) * cum[-1]) & (r > 0))[0]
            nxt = int(over[0]) if over.size else int(np.nonzero(r > 0)[0][-1])
    tokens = np.full(n + 1, -1, dtype=np.int32)
    tokens[:a] = drafts[:a]
    tokens[a] = nxt
    return tokens, a


