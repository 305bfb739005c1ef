"""Operators over device memory whose speed is tracked: the quantised KV cache,
attention over it, and the verification of drafted tokens.

Four kinds of case, each a call that a serving program makes:

  store   KvCache.write of new tokens' key and value rows, and KvCache.read of
          the rows they became (what the cache holds, as the values it stands
          for).
  read    KvCache.read of a history.
  attend  KvCache.attention of new tokens (their rows already in the cache):
          single tokens, drafted tokens, prompts, a shared prefix.
  verify  HipBackend.verify_drafts: which drafted tokens stand, and the token
          that follows them.

With `own` false the same results come from elementary torch operations.
"""
import math

import torch

own = False

FAR = 1 << 30   # a window that hides nothing


def listed():
    return [
        # The smallest model's single token on its way into the cache: all latency.
        dict(name="store_token_tiny", kind="store", batch=1, tokens=1, kv_heads=8, head_dim=64, k="q8_0", v="q8_0",
             longest=100, ragged=False),
        # The 7B shape's longest prompt chunk, behind an odd number of positions.
        dict(name="store_prompt_7b", kind="store", batch=1, tokens=2048, kv_heads=8, head_dim=128, k="q8_0", v="q8_0",
             longest=1003, ragged=False),
        # Seven sessions of the 1B shape read back from a 4-bit cache, each of its own length.
        dict(name="read_ragged_1b", kind="read", batch=7, tokens=1500, kv_heads=8, head_dim=64, k="q4_0", v="q4_0",
             longest=0, ragged=True),
        # One long session of the 7B shape read back.
        dict(name="read_long_7b", kind="read", batch=1, tokens=32768, kv_heads=8, head_dim=128, k="q8_0", v="q8_0",
             longest=0, ragged=False),
        # The smallest model early in a chat: one token over a hundred positions.
        dict(name="attend_token_tiny", kind="attend", batch=1, tokens=1, heads=8, kv_heads=8, head_dim=64, k="q8_0",
             v="q8_0", longest=100, ragged=False, prefix=0, window=0),
        # The 7B shape's decode step at the end of a 4096-token context.
        dict(name="attend_token_7b_4096", kind="attend", batch=1, tokens=1, heads=32, kv_heads=8, head_dim=128,
             k="q8_0", v="q8_0", longest=4095, ragged=False, prefix=0, window=0),
        # Sixteen chats of the 1B shape, from short to 8000 tokens, 8-bit keys and 4-bit values.
        dict(name="attend_batch_1b", kind="attend", batch=16, tokens=1, heads=32, kv_heads=8, head_dim=64, k="q8_0",
             v="q4_0", longest=8000, ragged=True, prefix=0, window=0),
        # Up to five drafted tokens of four chats of the Phi-3-mini shape (a kv head per head) under its sliding window.
        dict(name="attend_drafts_phi", kind="attend", batch=4, tokens=5, heads=32, kv_heads=32, head_dim=96, k="q8_0",
             v="q8_0", longest=2400, ragged=True, prefix=0, window=2047),
        # Thirty-two continuations of one long prompt of the 7B shape, each with a short tail of its own.
        dict(name="attend_prefix_7b", kind="attend", batch=32, tokens=1, heads=32, kv_heads=8, head_dim=128, k="q8_0",
             v="q8_0", longest=250, ragged=True, prefix=6000, window=0),
        # The 7B shape's longest prompt chunk.
        dict(name="attend_prompt_7b", kind="attend", batch=1, tokens=2048, heads=32, kv_heads=8, head_dim=128,
             k="q8_0", v="q8_0", longest=0, ragged=False, prefix=0, window=0),
        # Four tokens looked up in the prompt (no draft model) for one chat over the 7B shape's vocabulary.
        dict(name="verify_lookup_7b", kind="verify", batch=1, drafts=4, vocab=32000, draft_model=False, ragged=False),
        # A draft model's five tokens for each of sixteen chats over the 1B shape's vocabulary.
        dict(name="verify_batch_1b", kind="verify", batch=16, drafts=5, vocab=128256, draft_model=True, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _drawn(rng):
    kind = rng.choice(["store", "read", "attend", "attend", "attend", "verify"])
    if kind == "verify":
        return dict(kind=kind, batch=_log_int(rng, 1, 32), drafts=rng.randint(1, 8), vocab=_log_int(rng, 1000, 160000),
                    draft_model=rng.random() < 0.6, ragged=rng.random() < 0.5)
    case = dict(kind=kind, batch=_log_int(rng, 1, 32), kv_heads=rng.choice([1, 2, 4, 8, 8, 32]),
                head_dim=rng.choice([64, 96, 128, 128, 256]), k=rng.choice(["q8_0", "q4_0"]),
                v=rng.choice(["q8_0", "q4_0"]), ragged=rng.random() < 0.6)
    if kind == "store":
        return dict(case, tokens=_log_int(rng, 1, 2048), longest=rng.randint(0, 4000))
    if kind == "read":
        return dict(case, tokens=_log_int(rng, 1, 32768), longest=0)
    many = rng.random() < 0.3   # prompts, else single and drafted tokens
    return dict(case, heads=case["kv_heads"] * rng.choice([1, 2, 4, 4, 7, 8]),
                tokens=_log_int(rng, 16, 2048) if many else rng.choice([1, 1, rng.randint(2, 8)]),
                longest=_log_int(rng, 1, 32000), prefix=_log_int(rng, 16, 16000) if rng.random() < 0.3 else 0,
                window=_log_int(rng, 8, 8000) if rng.random() < 0.25 else 0)


def draw(rng):
    most = [work(c) for c in listed()]
    most = {m: max(w[m] for w in most) for m in most[0]}
    while True:
        case = _drawn(rng)
        w = work(case)
        scores = case["batch"] * case.get("heads", 0) * case["tokens"] * (case["longest"] + case["tokens"] + case["prefix"]) \
            if case["kind"] == "attend" else 0
        if all(w[m] <= most[m] for m in most) and scores <= 200_000_000:
            return case


# ------------------------------------------------------------------ inputs --

def _rows(case):
    """Each sequence's first new position and its number of new tokens: part of the case, not of its seed."""
    b = case["batch"]
    if not case["ragged"]:
        return [case["longest"]] * b, [case["tokens"]] * b
    part = [(0.381966 + 0.618034 * i) % 1.0 for i in range(b)]
    if case["kind"] == "read":
        return [0] * b, [max(1, round(case["tokens"] * x)) for x in part]
    starts = [int(case["longest"] * x) for x in part]
    return starts, [case["tokens"] - i % min(case["tokens"], 4) for i in range(b)]


def _counts(case):
    return [case["drafts"] - (i % (case["drafts"] + 1) if case["ragged"] else 0) for i in range(case["batch"])]


def _shape(case, rows):
    return (case["batch"], rows, case["kv_heads"], case["head_dim"])


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _keys(g, *shape):
    """Keys as models have them: a few dimensions of each head are several times the others."""
    x = _normal(g, *shape)
    x[..., 3::29] *= 4.0
    return x


def _capacity(case):
    starts, counts = _rows(case)
    return max(s + c for s, c in zip(starts, counts))


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _slots(case):
    return [case["batch"] - 1 - i for i in range(case["batch"])]


def _cache_data(case, seed):
    """New rows (store), or all rows of a history (read, attend); the prefix's rows; queries."""
    g = _generator(seed)
    d = {}
    n = case["tokens"] if case["kind"] == "store" else _capacity(case)
    d["k"], d["v"] = _keys(g, *_shape(case, n)), _normal(g, *_shape(case, n))
    if case["kind"] == "attend":
        d["q"] = _normal(g, case["batch"], case["tokens"], case["heads"], case["head_dim"]) * 1.3
        if case["prefix"]:
            shape = (1, case["prefix"], case["kv_heads"], case["head_dim"])
            d["pk"], d["pv"] = _keys(g, *shape), _normal(g, *shape)
    return d


def _verify_data(case, seed):
    """Logits with a broad bulk and some favourites; the draft model's are near the target's; tokens drawn from it."""
    g = _generator(seed)
    b, n, vocab = case["batch"], case["drafts"], case["vocab"]
    target = _normal(g, b, n + 1, vocab) * 1.5
    top = torch.randint(vocab, (b, n + 1, 40), generator=g, device="cuda")
    target.scatter_add_(2, top, 4.0 + 5.0 * torch.rand(b, n + 1, 40, generator=g, device="cuda"))
    draft = target[:, :n] + 0.7 * _normal(g, b, n, vocab)
    probs = torch.softmax((draft if case["draft_model"] else 2.0 * target[:, :n]) / 0.8, -1)
    at = torch.rand(b, n, 1, generator=g, device="cuda")
    tokens = (probs.double().cumsum(-1) <= at).sum(-1).clamp(max=vocab - 1).to(torch.int32)
    return dict(target=target.contiguous(), draft=draft.contiguous() if case["draft_model"] else None, tokens=tokens,
                uniforms=torch.rand(b, n + 1, generator=g, device="cuda"),
                temperature=torch.tensor(0.8).item())   # the 32-bit number that an option holds


_shared = {}


def _backend():
    """The one backend that a program creates at its start."""
    if "backend" not in _shared:
        from dotllm_amd import HipBackend
        _shared["backend"] = HipBackend()
    return _shared["backend"]


def _own_cache(case, slots, capacity):
    from dotllm_amd import KvCache, _lib
    return KvCache(_backend(), slots=slots, kv_heads=case["kv_heads"], head_dim=case["head_dim"], capacity=capacity,
                   k_type=getattr(_lib, case["k"].upper()), v_type=getattr(_lib, case["v"].upper()))


def _plain_cache(case, slots, capacity):
    kind = dict(dtype=torch.int8, device="cuda")
    scale = dict(dtype=torch.float16, device="cuda")
    shape = (slots, case["kv_heads"], capacity, case["head_dim"])
    blocks = shape[:3] + (case["head_dim"] // 32,)
    return dict(k=torch.zeros(shape, **kind), v=torch.zeros(shape, **kind), kd=torch.zeros(blocks, **scale),
                vd=torch.zeros(blocks, **scale))


def prepare(case, seed):
    if case["kind"] == "verify":
        s = dict(_verify_data(case, seed), case=case, counts=_ints(_counts(case)))
        s["tokens_out"] = torch.empty(case["batch"], case["drafts"] + 1, dtype=torch.int32, device="cuda")
        s["accepted_out"] = torch.empty(case["batch"], dtype=torch.int32, device="cuda")
        if own:
            s["workspace"] = _backend().verify_workspace(case["batch"], case["drafts"], case["vocab"])
        return s
    data = _cache_data(case, seed)
    starts, counts = _rows(case)
    s = dict(case=case, slots=_ints(_slots(case)), starts=_ints(starts), counts=_ints(counts))
    n = case["tokens"]
    if case["kind"] != "attend":   # rows past a sequence's count are never written: zeros on both sides
        s["k_out"] = torch.zeros(_shape(case, n), dtype=torch.float32, device="cuda")
        s["v_out"] = torch.zeros(_shape(case, n), dtype=torch.float32, device="cuda")
    if case["kind"] == "store":
        s["k"], s["v"] = data["k"], data["v"]
    if case["kind"] == "attend":
        s["q"], s["out"] = data["q"], torch.zeros_like(data["q"])
    torch.cuda.synchronize()
    if own:
        s["cache"] = _own_cache(case, case["batch"], _capacity(case))
        s["tokens"] = s["cache"].batch(n, s["slots"], s["starts"], s["counts"])
    else:
        s["cache"] = _plain_cache(case, case["batch"], _capacity(case))
    if case["kind"] != "store":
        _fill(s["cache"], data["k"], data["v"], case, s["slots"])
    if case["kind"] == "attend":
        s["prefix"] = None
        if case["prefix"]:
            s["prefix"] = _own_cache(case, 1, case["prefix"]) if own else _plain_cache(case, 1, case["prefix"])
            _fill(s["prefix"], data["pk"], data["pv"], case, _ints([0]))
        if own:
            s["workspace"] = s["cache"].attention_workspace(case["heads"], case["batch"], n, s["prefix"] is not None)
    torch.cuda.synchronize()
    return s


def _fill(cache, k, v, case, slots):
    """A history's rows, written whole (those past a sequence's end are never seen)."""
    zero = torch.zeros_like(slots)
    if own:
        torch.cuda.synchronize()
        cache.write(k, v, cache.batch(k.shape[1], slots, zero))
        torch.cuda.synchronize()
    else:
        _plain_write(cache, k, v, slots, zero, torch.full_like(slots, k.shape[1]), case)


def run(state):
    case = state["case"]
    if not own:
        return _PLAIN[case["kind"]](state)
    if case["kind"] == "verify":
        _backend().verify_drafts(state["target"], state["tokens"], state["uniforms"], state["tokens_out"],
                                 state["accepted_out"], draft=state["draft"], counts=state["counts"],
                                 temperature=state["temperature"], workspace=state["workspace"])
        return state["tokens_out"], state["accepted_out"]
    cache, tokens = state["cache"], state["tokens"]
    if case["kind"] == "attend":
        cache.attention(state["q"], state["out"], tokens, prefix=state["prefix"], prefix_len=case["prefix"],
                        window=case["window"], workspace=state["workspace"])
        return state["out"]
    if case["kind"] == "store":
        cache.write(state["k"], state["v"], tokens)
    cache.read(state["k_out"], state["v_out"], tokens)
    return state["k_out"], state["v_out"]


# -------------------------------------------------------------- plain forms --

def _round(x):
    """To the nearest integer, halves away from zero."""
    t = torch.trunc(x)
    return t + torch.sign(x) * ((x - t).abs() >= 0.5)


def _quantize(x, kind):
    """Blocks of 32 along the last dimension: integers and 16-bit scales, as the package's quantiser makes them."""
    b = x.unflatten(-1, (-1, 32))
    mag = b.abs()
    top = mag.amax(-1, keepdim=True)
    if kind == "q8_0":
        d = (top / torch.full_like(top, 127.0)).half()   # a quotient: a division by a number is a product on the device
    else:   # the signed value of the first largest magnitude becomes -8
        lane = torch.arange(32, device=x.device)
        first = torch.where(mag == top, lane, 32).amin(-1, keepdim=True)
        d = (b.gather(-1, first) / -8.0).half()
    step = d.float()
    q = torch.where(step == 0, torch.zeros_like(b), _round(b / torch.where(step == 0, torch.ones_like(step), step)))
    q = q.clamp(-127, 127) if kind == "q8_0" else q.clamp(-8, 7)
    return q.flatten(-2).to(torch.int8), d.squeeze(-1)


def _place(slots, starts, counts, tokens):
    """Slot, position and (sequence, token) of every row that is there."""
    i = torch.arange(tokens, device=slots.device)
    b, t = torch.nonzero(i[None, :] < counts[:, None], as_tuple=True)
    return slots.long()[b], (starts.long()[b] + t), b, t


def _plain_write(cache, k, v, slots, starts, counts, case):
    slot, pos, b, t = _place(slots, starts, counts, k.shape[1])
    kq, kd = _quantize(k[b, t], case["k"])
    vq, vd = _quantize(v[b, t], case["v"])
    cache["k"][slot, :, pos], cache["kd"][slot, :, pos] = kq, kd
    cache["v"][slot, :, pos], cache["vd"][slot, :, pos] = vq, vd


def _values(q, d):
    return (q.float().unflatten(-1, (-1, 32)) * d.float().unsqueeze(-1)).flatten(-2)


def _plain_read(state):
    cache = state["cache"]
    slot, pos, b, t = _place(state["slots"], state["starts"], state["counts"], state["case"]["tokens"])
    state["k_out"][b, t] = _values(cache["k"][slot, :, pos], cache["kd"][slot, :, pos])
    state["v_out"][b, t] = _values(cache["v"][slot, :, pos], cache["vd"][slot, :, pos])
    return state["k_out"], state["v_out"]


def _plain_store(state):
    _plain_write(state["cache"], state["k"], state["v"], state["slots"], state["starts"], state["counts"],
                 state["case"])
    return _plain_read(state)


def _plain_attend(state):
    case, cache, prefix = state["case"], state["cache"], state["prefix"]
    b, n, heads, hd = state["q"].shape
    kvh, most, first = case["kv_heads"], cache["k"].shape[2], case["prefix"]
    window = case["window"] or FAR
    slots = state["slots"].long()
    # rows of a kv head: its query heads of every token
    q = state["q"].reshape(b, n, kvh, heads // kvh, hd).permute(0, 2, 1, 3, 4).reshape(b, kvh, -1, hd) / math.sqrt(hd)
    own_k = _values(cache["k"][slots], cache["kd"][slots])
    own_v = _values(cache["v"][slots], cache["vd"][slots])
    scores = q @ own_k.transpose(-1, -2)
    token = torch.arange(n, device=q.device).repeat_interleave(heads // kvh)
    at = state["starts"][:, None, None] + token[None, :, None]
    key = torch.arange(most, device=q.device)
    scores = scores.masked_fill(((key > at) | (key <= at - window))[:, None], -math.inf)
    if prefix is not None:
        pk, pv = _values(prefix["k"][0], prefix["kd"][0]), _values(prefix["v"][0], prefix["vd"][0])
        shared = q.transpose(0, 1).reshape(kvh, -1, hd) @ pk.transpose(-1, -2)
        shared = shared.reshape(kvh, b, -1, first).transpose(0, 1)
        hidden = torch.arange(first, device=q.device) - first <= at - window
        scores = torch.cat([shared.masked_fill(hidden[:, None], -math.inf), scores], -1)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = e[..., first:] @ own_v
    if prefix is not None:
        shared = e[..., :first].transpose(0, 1).reshape(kvh, -1, first) @ pv
        out = out + shared.reshape(kvh, b, -1, hd).transpose(0, 1)
    out = (out / e.sum(-1, keepdim=True)).reshape(b, kvh, n, -1, hd).transpose(1, 2).reshape(b, n, heads, hd)
    there = torch.arange(n, device=q.device)[None, :] < state["counts"][:, None]
    state["out"].copy_(torch.where(there[:, :, None, None], out, torch.zeros_like(out)))
    return state["out"]


def _plain_verify(state):
    """In 64 bits: tokens next to a border of the distribution."""
    n, counts = state["tokens"].shape[1], state["counts"].long()
    scaled = state["target"].double() / state["temperature"]
    e = torch.exp(scaled - scaled.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    at = state["tokens"].long().unsqueeze(-1)
    if state["draft"] is None:
        q = torch.zeros_like(p[:, :n]).scatter_(-1, at, 1.0)
    else:
        scaled = state["draft"].double() / state["temperature"]
        e = torch.exp(scaled - scaled.amax(-1, keepdim=True))
        q = e / e.sum(-1, keepdim=True)
    u = state["uniforms"].double()
    stands = u[:, :n] * q.gather(-1, at).squeeze(-1) < p[:, :n].gather(-1, at).squeeze(-1)
    lane = torch.arange(n + 1, device=p.device)
    accepted = (stands & (lane[:n] < counts[:, None])).long().cumprod(-1).sum(-1)
    rows = torch.arange(p.shape[0], device=p.device)
    p_at = p[rows, accepted]
    q_at = torch.where((accepted < counts)[:, None], q[rows, accepted.clamp(max=n - 1)], torch.zeros_like(p_at))
    r = (p_at - q_at).clamp(min=0.0)
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, p_at)
    cum = r.cumsum(-1)
    token = (cum <= u[:, n:] * cum[:, -1:]).sum(-1).clamp(max=p.shape[-1] - 1)
    drafted = torch.cat([state["tokens"], state["tokens"][:, :1]], -1).long()
    out = torch.where(lane < accepted[:, None], drafted,
                      torch.where(lane == accepted[:, None], token[:, None], torch.full_like(drafted, -1)))
    state["tokens_out"].copy_(out)
    state["accepted_out"].copy_(accepted)
    return state["tokens_out"], state["accepted_out"]


_PLAIN = {"store": _plain_store, "read": _plain_read, "attend": _plain_attend, "verify": _plain_verify}


# ---------------------------------------------------------- necessary work ----

_BYTES = {"q8_0": 34 / 32, "q4_0": 18 / 32}


def work(case):
    if case["kind"] == "verify":
        rows = sum(n + 1 + (n if case["draft_model"] else 0) for n in _counts(case))
        return {"bytes": 4.0 * rows * case["vocab"], "flops": 4.0 * rows * case["vocab"]}
    starts, counts = _rows(case)
    width = case["kv_heads"] * case["head_dim"]
    held = _BYTES[case["k"]] + _BYTES[case["v"]]
    if case["kind"] != "attend":   # fp32 rows in (store), quantised rows, fp32 rows out
        n = sum(counts)
        return {"bytes": n * width * (held + (16.0 if case["kind"] == "store" else 8.0)),
                "flops": n * width * (8.0 if case["kind"] == "store" else 2.0)}
    window, first = case["window"] or FAR, case["prefix"]
    pairs = rows = 0
    low = first   # the first prefix position that some query sees
    for s, c in zip(starts, counts):
        seen = 0
        for i in range(c):
            here = min(s + i + 1, window)
            before = min(first, max(0, window - (s + i + 1)))
            pairs += here + before
            low = min(low, first - before)
            seen = max(seen, here + i if window < FAR else here)
        rows += min(seen, s + c)
    n = sum(counts)
    return {"bytes": (rows + first - low) * width * held + 8.0 * n * case["heads"] * case["head_dim"],
            "flops": 4.0 * pairs * case["heads"] * case["head_dim"]}


# --------------------------------------------- the same results in 64 bits --

def _held64(x, kind):
    """What the cache holds for x, in 64 bits: the format rounds its scale to 16 bits by way of 32, and each
    quotient to 32 bits before it becomes an integer."""
    blocks = x.double().reshape(*x.shape[:-1], -1, 32)
    if kind == "q8_0":
        scale = (blocks.abs().max(-1).values / torch.full((), 127.0, dtype=torch.float64, device=x.device)).float().half().double()
        low, high = -127, 127
    else:
        most = (blocks.abs() == blocks.abs().max(-1, keepdim=True).values)
        which = (most * torch.arange(32, 0, -1, device=x.device)).argmax(-1, keepdim=True)
        scale = (blocks.gather(-1, which).squeeze(-1) / -8).float().half().double()
        low, high = -8, 7
    scale = scale.unsqueeze(-1)
    ratio = torch.nan_to_num((blocks / scale).float().double(), 0.0, 0.0, 0.0)
    near = torch.sign(ratio) * torch.floor(ratio.abs() + 0.5)
    return (near.clamp(low, high) * scale).reshape(x.shape)


def exact(case, seed):
    if case["kind"] == "verify":
        return None   # token ids and counts
    data = _cache_data(case, seed)
    starts, counts = _rows(case)
    if case["kind"] != "attend":
        got = []
        for x, kind in ((data["k"], case["k"]), (data["v"], case["v"])):
            y = _held64(x, kind)
            out = torch.zeros(_shape(case, case["tokens"]), dtype=torch.float64, device="cuda")
            for b, c in enumerate(counts):
                out[b, :c] = y[b, :c]
            got.append(out.cpu())
        return tuple(got)
    heads, kvh, hd, first = case["heads"], case["kv_heads"], case["head_dim"], case["prefix"]
    out = torch.zeros(data["q"].shape, dtype=torch.float64, device="cuda")
    window = case["window"] or FAR
    for b, (s, c) in enumerate(zip(starts, counts)):
        k, v = _held64(data["k"][b, :s + c], case["k"]), _held64(data["v"][b, :s + c], case["v"])
        if first:
            k = torch.cat([_held64(data["pk"][0], case["k"]), k])
            v = torch.cat([_held64(data["pv"][0], case["v"]), v])
        where = torch.arange(first + s + c, device="cuda")
        here = first + s + torch.arange(c, device="cuda")
        seen = (where[None, :] <= here[:, None]) & (where[None, :] > here[:, None] - window)
        for h in range(heads):
            j = h // (heads // kvh)
            score = data["q"][b, :c, h].double() @ k[:, j].t().contiguous() / math.sqrt(hd)
            score = torch.where(seen, score, torch.full_like(score, -math.inf))
            weight = torch.softmax(score, -1)
            out[b, :c, h] = weight @ v[:, j].contiguous()
    return out.cpu()
