"""The cases of the operators around a drafted continuation: what a program does
that lets a small model draft several tokens and has the large one check them
in one pass.

Four kinds of case:

- "append": the drafted rows' queries and keys normed and rotated, keys and
  values written to a cache of several sequences in its own format, and the
  rows just written read back as the values that they stand for.
- "read": everything a cache holds, as f32 rows.
- "attend": the rows' attention over the cache, each row over the positions
  before the draft and over its own ancestors among the drafted rows (a chain:
  over the rows before it).
- "score": log probabilities of given tokens, the entropy of each row's
  distribution and its most likely tokens.

Sequences have their own lengths and row counts; rows beyond a sequence's
count stay as they were. Formats of a cache: "f32", "f16", and "q8": one byte
per element and one f32 scale per position and head,
scale = max |x| / 127 rounded to f32, byte = x / scale rounded to even.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EPS = 1e-6
ELEMENT = {"f32": 4, "f16": 2, "q8": 1}


def listed():
    return [
        # one token of one sentence: the talker's own step, all latency
        dict(name="append_token", op="append", n=1, rows=1, len=300, heads=16, kv_heads=8,
             head_dim=128, fmt="f32", tree=False, rot_dim=128, interleaved=False,
             scaling="plain", theta=1e6),
        # a server's drafts: 16 sequences of long text, positions past those trained on
        dict(name="append_trees_q8", op="append", n=16, rows=31, len=20000, heads=16, kv_heads=8,
             head_dim=128, fmt="q8", tree=True, rot_dim=128, interleaved=False,
             scaling="yarn", theta=1e6),
        # prompts of ragged length, half of each head rotated in neighbouring pairs
        dict(name="append_prompts_f16", op="append", n=6, rows=1021, len=4000, heads=32,
             kv_heads=8, head_dim=128, fmt="f16", tree=False, rot_dim=64, interleaved=True,
             scaling="linear", theta=1e4),
        # a short sentence's cache handed on
        dict(name="read_short_f16", op="read", n=1, len=37, kv_heads=8, head_dim=128, fmt="f16"),
        # the caches of a server's sequences handed on
        dict(name="read_q8", op="read", n=8, len=4099, kv_heads=8, head_dim=128, fmt="q8"),
        # one token of one sentence over an f32 cache
        dict(name="attend_token", op="attend", n=1, rows=1, len=171, heads=16, kv_heads=8,
             head_dim=128, fmt="f32", tree=False),
        # one token of each of a server's 32 sentences
        dict(name="attend_tokens_q8", op="attend", n=32, rows=1, len=2048, heads=16, kv_heads=8,
             head_dim=128, fmt="q8", tree=False),
        # one drafted tree over a long context
        dict(name="attend_tree_f16", op="attend", n=1, rows=27, len=12289, heads=16, kv_heads=8,
             head_dim=128, fmt="f16", tree=True),
        # wide trees of 12 long sequences, four query heads to a key head
        dict(name="attend_trees_q8", op="attend", n=12, rows=64, len=8000, heads=32, kv_heads=8,
             head_dim=128, fmt="q8", tree=True),
        # one code chosen from a codebook's distribution
        dict(name="score_token", op="score", rows=1, vocab=2048, dtype="f32", tokens=1, top_k=5,
             suppressed=0.0),
        # drafted text tokens over a text vocabulary
        dict(name="score_text", op="score", rows=40, vocab=151936, dtype="f32", tokens=1,
             top_k=20, suppressed=0.0),
        # a long sentence's codes rescored, four candidates each, a part of the codes ruled out
        dict(name="score_codes", op="score", rows=1021, vocab=8191, dtype="bf16", tokens=4,
             top_k=3, suppressed=0.1),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "append", "attend", "attend", "attend", "score", "score", "read"))
    if op == "score":
        vocab = _spread(rng, 200, 152000)
        return dict(op=op, rows=_spread(rng, 1, max(1, min(1200, 6000000 // vocab))), vocab=vocab,
                    dtype=rng.choice(("f32", "bf16")), tokens=rng.choice((1, 1, 2, 5)),
                    top_k=rng.choice((0, 1, 5, 10, 33, 64)),
                    suppressed=rng.choice((0.0, 0.0, 0.3)))
    heads, kv_heads = rng.choice(((16, 8), (16, 8), (8, 8), (32, 8), (6, 2), (28, 4), (8, 1)))
    fmt = rng.choice(("f32", "f16", "q8", "q8"))
    hd = rng.choice((128, 128, 64))
    if op == "read":
        return dict(op=op, n=_spread(rng, 1, 16), len=_spread(rng, 1, 2000), kv_heads=kv_heads,
                    head_dim=hd, fmt=fmt)
    tree = rng.random() < 0.6
    if op == "append":
        n = _spread(rng, 1, 24)
        return dict(op=op, n=n, rows=_spread(rng, 1, 64 if tree else max(2, 2000 // n)),
                    len=0 if rng.random() < 0.1 else _spread(rng, 1, 16000), heads=heads, kv_heads=kv_heads, head_dim=hd,
                    fmt=fmt, tree=tree, rot_dim=rng.choice((hd, hd, hd // 2, hd // 4, 6)),
                    interleaved=rng.random() < 0.4,
                    scaling=rng.choice(("plain", "linear", "yarn", "bands")),
                    theta=rng.choice((1e4, 1e6)))
    rows = rng.choice((1, 1, _spread(rng, 2, 64), 0 if tree else _spread(rng, 2, 200)))
    rows = rows or _spread(rng, 2, 64)
    n = _spread(rng, 1, 24)
    most = min(16000, 40000 // n, int(3e6) // (n * rows))
    length = 0 if rng.random() < 0.1 else _spread(rng, 1, max(2, most))
    return dict(op=op, n=n, rows=rows, len=length, heads=heads, kv_heads=kv_heads, head_dim=hd,
                fmt=fmt, tree=tree and rows <= 64)


def _lens(case):
    """Lengths of the sequences, longest first: down to a quarter of the longest."""
    n, top = case["n"], case["len"]
    return [top - (3 * top * i) // (4 * max(1, n - 1)) if n > 1 else top for i in range(n)]


def _counts(case):
    """Drafted rows of the sequences: from all of them down to a few."""
    n, rows = case["n"], case["rows"]
    return [max(1, rows - rows * i // n) for i in range(n)]


# ---------------------------------------------------------------------------
# rotary frequencies, in 64 bits


SCALING = {
    "plain": None,
    "linear": dict(kind="linear", factor=2.0),
    "yarn": dict(kind="yarn", factor=4.0, original=8192, beta_fast=32.0, beta_slow=1.0),
    "bands": dict(kind="bands", factor=8.0, original=8192, low=1.0, high=4.0),
}


def _frequencies(case):
    """(angle per position of each rotated pair, factor on cosine and sine)."""
    d, theta, s = case["rot_dim"], case["theta"], SCALING[case["scaling"]]
    i = torch.arange(d // 2, dtype=torch.float64, device="cuda")
    f = theta ** (-2.0 * i / d)
    if s is None:
        return f, 1.0
    if s["kind"] == "linear":
        return f / s["factor"], 1.0
    if s["kind"] == "yarn":
        turn = lambda b: d * math.log(s["original"] / (b * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(0, math.floor(turn(s["beta_fast"]))), min(d - 1, math.ceil(turn(s["beta_slow"])))
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / s["factor"] * ramp + f * (1 - ramp), 0.1 * math.log(s["factor"]) + 1.0
    turns = s["original"] * f / (2 * math.pi)
    mix = ((turns - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
    return f * mix + f / s["factor"] * (1 - mix), 1.0


# ---------------------------------------------------------------------------
# inputs, from the seed alone


def _gen(seed, part):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + part) % (1 << 62))
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    """The case's inputs: what both forms and exact() start from."""
    host = np.random.RandomState(int(seed) % (1 << 31))
    op = case["op"]
    x = {}
    if op == "score":
        g = _gen(seed, 1)
        logits = _normal(g, case["rows"], case["vocab"]) * 2.5
        if case["suppressed"]:
            off = torch.rand(case["vocab"], generator=g, device="cuda") < case["suppressed"]
            logits = logits.masked_fill(off, -math.inf)
        x["logits"] = logits.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        x["tokens"] = _ints(host.randint(0, case["vocab"], (case["rows"], case["tokens"])))
        return x
    n, kvh, hd = case["n"], case["kv_heads"], case["head_dim"]
    order = host.permutation(n)
    x["lens"] = _ints(np.array(_lens(case))[order])
    if op == "read":
        # keys with the outlying channels that trained ones have
        wide = torch.exp(0.5 * _normal(_gen(seed, 2), kvh, hd))
        x["k"] = _normal(_gen(seed, 3), n, case["len"], kvh, hd) * wide
        x["v"] = _normal(_gen(seed, 4), n, case["len"], kvh, hd)
        return x
    rows, h = case["rows"], case["heads"]
    x["counts"] = _ints(np.array(_counts(case))[host.permutation(n)])
    # a node's parent: most often one of the last few, at times none of them
    back = host.geometric(0.4, (n, rows))
    parents = np.maximum(np.arange(rows)[None, :] - back, -1) if case["tree"] else \
        np.broadcast_to(np.arange(rows)[None, :] - 1, (n, rows))
    x["parents"] = _ints(np.ascontiguousarray(parents))
    if op == "append":
        x["qkv"] = _normal(_gen(seed, 5), n, rows, (h + 2 * kvh) * hd)
        x["q_norm"] = 1 + 0.1 * _normal(_gen(seed, 6), hd)
        x["k_norm"] = torch.exp(0.5 * _normal(_gen(seed, 7), hd))
        return x
    wide = torch.exp(0.5 * _normal(_gen(seed, 2), kvh, hd))
    x["q"] = _normal(_gen(seed, 5), n, rows, h, hd)
    x["k"] = _normal(_gen(seed, 3), n, case["len"] + rows, kvh, hd) * wide
    x["v"] = _normal(_gen(seed, 4), n, case["len"] + rows, kvh, hd)
    return x


# ---------------------------------------------------------------------------
# a cache in its plain form: [sequence][head][position][element], one position
# more than it has, where rows go that are not stored


def _stored(rows, fmt):
    """f32 rows as the format holds them: (elements, scales)."""
    if fmt != "q8":
        return rows.to(torch.float16 if fmt == "f16" else torch.float32), None
    wide = rows.double()
    scale = (wide.abs().amax(-1, keepdim=True) / 127).float()
    return torch.round(wide / scale.double()).to(torch.int8), scale


def _plain_cache(case, positions):
    n, kvh, hd, fmt = case["n"], case["kv_heads"], case["head_dim"], case["fmt"]
    kind = {"f32": torch.float32, "f16": torch.float16, "q8": torch.int8}[fmt]
    make = lambda w, t: torch.zeros(n, kvh, positions + 1, w, device="cuda", dtype=t)  # noqa: E731
    return {"k": make(hd, kind), "v": make(hd, kind), "ks": make(1, torch.float32),
            "vs": make(1, torch.float32)}


def _put(cache, case, k, v, slots):
    at = torch.arange(case["n"], device="cuda")[:, None]
    ke, ks = _stored(k, case["fmt"])
    ve, vs = _stored(v, case["fmt"])
    cache["k"][at, :, slots] = ke
    cache["v"][at, :, slots] = ve
    if case["fmt"] == "q8":
        cache["ks"][at, :, slots] = ks
        cache["vs"][at, :, slots] = vs


def _values(cache, case, part, slots):
    """Rows [sequence][row][head][element] of the cache, in f32."""
    at = torch.arange(case["n"], device="cuda")[:, None]
    rows = cache[part][at, :, slots].float()
    return rows * cache[part + "s"][at, :, slots] if case["fmt"] == "q8" else rows


# ---------------------------------------------------------------------------


def _package():
    path = os.path.join(ROOT, "mormot2-qwen-tts_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import q3h
    return q3h


def _own_cache(case, positions):
    q3h = _package()
    dev = q3h.Device(0)
    fmt = {"f32": q3h.KV_F32, "f16": q3h.KV_F16, "q8": q3h.KV_Q8}[case["fmt"]]
    return dev, q3h.Cache(dev, case["n"], case["kv_heads"], case["head_dim"], positions, fmt)


def _own_rope(case, dev, positions):
    q3h = _package()
    return q3h.Rope(dev, case["head_dim"], positions, case["theta"], rot_dim=case["rot_dim"],
                    interleaved=case["interleaved"], scaling=SCALING[case["scaling"]])


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": case, "x": x}
    op = case["op"]
    if op == "score":
        if own:
            state["dev"] = _package().Device(0)
        return state
    positions = case["len"] + (0 if op == "read" else case["rows"])
    n, kvh, hd = case["n"], case["kv_heads"], case["head_dim"]
    if own:
        state["dev"], state["cache"] = _own_cache(case, positions)
    else:
        state["cache"] = _plain_cache(case, positions)
    rows = case["len"] if op == "read" else case["rows"]
    if op == "append":
        if own:
            state["rope"] = _own_rope(case, state["dev"], positions)
        else:
            state["rope"] = _frequencies(case)
    else:
        # the cache as earlier appends left it
        held = x["lens"] + (0 if op == "read" else x["counts"])
        if own:
            state["cache"].append(x["k"], x["v"], torch.zeros_like(held), counts=held)
        else:
            slots = torch.arange(positions, device="cuda")[None, :].expand(n, -1)
            slots = torch.where(slots < held[:, None], slots, positions)
            _put(state["cache"], case, x["k"], x["v"], slots)
        del x["k"], x["v"]
    # the buffers of a program's outputs, rows of no sequence zero
    if op != "read":
        state["q_out"] = torch.zeros(n, rows, case["heads"], hd, device="cuda")
    if op != "attend":
        state["k_out"] = torch.zeros(n, rows, kvh, hd, device="cuda")
        state["v_out"] = torch.zeros(n, rows, kvh, hd, device="cuda")
    return state


# ---------------------------------------------------------------------------
# the framework's operators


def _run_own(state):
    case, x = state["case"], state["x"]
    op = case["op"]
    if op == "score":
        return _package().token_logprobs(state["dev"], x["logits"], x["tokens"],
                                         top_k=case["top_k"])
    cache = state["cache"]
    if op == "read":
        cache.read(state["k_out"], state["v_out"], counts=x["lens"])
        return {"k": state["k_out"], "v": state["v_out"]}
    parents = x["parents"] if case["tree"] else None
    if op == "attend":
        cache.attend(x["q"], x["lens"], case["len"], out=state["q_out"], counts=x["counts"],
                     parents=parents)
        return {"out": state["q_out"]}
    h, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    q, k, v = x["qkv"].split((h * hd, kvh * hd, kvh * hd), dim=-1)
    cache.append(k, v, x["lens"], counts=x["counts"], parents=parents, q=q,
                 q_out=state["q_out"], rope=state["rope"], q_norm=x["q_norm"],
                 k_norm=x["k_norm"], eps=EPS)
    cache.read(state["k_out"], state["v_out"], starts=x["lens"], counts=x["counts"])
    return {"q": state["q_out"], "k": state["k_out"], "v": state["v_out"]}


# ---------------------------------------------------------------------------
# the plain forms


def _square(reach):
    return (reach @ reach).clamp(max=1)


def _ancestors(parents):
    """[sequence][row][row]: whether a row is the other one or comes after it on its path
    (of at most 64 rows: each squaring doubles the steps that are followed)."""
    rows = parents.shape[1]
    t = torch.arange(rows, device="cuda", dtype=torch.int32)
    step = ((parents[:, :, None] == t) | (t[:, None] == t)).float()
    return _square(_square(_square(_square(_square(_square(step)))))) > 0


def _depth(case, parents):
    if not case["tree"]:
        return torch.arange(case["rows"], device="cuda")[None, :]
    return _ancestors(parents).sum(-1) - 1


def _normed(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()


def _rotated(x, case, freq, pos):
    f, mag = freq
    angle = (pos.double()[:, :, None] * f)[:, :, None, :]
    cos, sin = angle.cos() * mag, angle.sin() * mag
    d = case["rot_dim"]
    r, rest = x[..., :d], x[..., d:]
    if case["interleaved"]:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :d // 2], r[..., d // 2:]
        r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((r, rest), -1).float()


def _run_append(state):
    case, x, cache = state["case"], state["x"], state["cache"]
    n, rows, h, kvh, hd = (case[k] for k in ("n", "rows", "heads", "kv_heads", "head_dim"))
    t = torch.arange(rows, device="cuda")[None, :]
    live = t < x["counts"][:, None]
    slots = torch.where(live, x["lens"][:, None] + t, case["len"] + rows)
    pos = x["lens"][:, None] + _depth(case, x["parents"])
    qkv = x["qkv"].view(n, rows, h + 2 * kvh, hd)
    q, k, v = qkv[:, :, :h].double(), qkv[:, :, h:h + kvh].double(), qkv[:, :, h + kvh:]
    q = _rotated(_normed(q, x["q_norm"]), case, state["rope"], pos)
    k = _rotated(_normed(k, x["k_norm"]), case, state["rope"], pos)
    _put(cache, case, k, v, slots)
    keep = live[:, :, None, None]
    return {"q": torch.where(keep, q, 0),
            "k": torch.where(keep, _values(cache, case, "k", slots), 0),
            "v": torch.where(keep, _values(cache, case, "v", slots), 0)}


def _run_read(state):
    case, x, cache = state["case"], state["x"], state["cache"]
    slots = torch.arange(case["len"], device="cuda")[None, :].expand(case["n"], -1)
    live = (slots < x["lens"][:, None])[:, :, None, None]
    return {"k": torch.where(live, _values(cache, case, "k", slots), 0),
            "v": torch.where(live, _values(cache, case, "v", slots), 0)}


def _run_attend(state):
    case, x, cache = state["case"], state["x"], state["cache"]
    n, rows, h, kvh, hd = (case[k] for k in ("n", "rows", "heads", "kv_heads", "head_dim"))
    positions, g = case["len"] + rows, h // kvh
    lens, counts = x["lens"][:, None, None], x["counts"][:, None, None]
    k, v = cache["k"][:, :, :positions].float(), cache["v"][:, :, :positions].float()
    if case["fmt"] == "q8":
        k, v = k * cache["ks"][:, :, :positions], v * cache["vs"][:, :, :positions]
    q = x["q"].view(n, rows, kvh, g, hd).permute(0, 2, 3, 1, 4).reshape(n, kvh, g * rows, hd)
    s = (q @ k.transpose(-1, -2)).view(n, kvh, g, rows, positions) * hd ** -0.5
    j = torch.arange(positions, device="cuda")[None, None, :]
    t = (j - lens).clamp(0, rows - 1)
    if case["tree"]:
        path = torch.gather(_ancestors(x["parents"]), 2, t.expand(-1, rows, -1).long())
    else:
        path = t <= torch.arange(rows, device="cuda")[None, :, None]
    sees = (j < lens) | (path & (j < lens + counts))
    s = s.masked_fill(~sees[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(n, kvh, g * rows, positions)
    out = (p @ v).view(n, kvh, g, rows, hd).permute(0, 3, 1, 2, 4).reshape(n, rows, h, hd)
    live = torch.arange(rows, device="cuda")[None, :] < x["counts"][:, None]
    return {"out": torch.where(live[:, :, None, None], out, 0)}


def _run_score(state):
    case, x = state["case"], state["x"]
    z = x["logits"].float()
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    logp = z - top - torch.log(total)
    entropy = -torch.where(e > 0, e / total * logp, 0).sum(-1)
    answer = {"logprobs": torch.gather(logp, 1, x["tokens"].long()), "entropy": entropy}
    if case["top_k"]:
        order = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :case["top_k"]]
        answer["top_ids"] = order.to(torch.int32)
        answer["top_logprobs"] = torch.gather(logp, 1, order)
    return answer


def run(state):
    if own:
        return _run_own(state)
    return {"append": _run_append, "read": _run_read, "attend": _run_attend,
            "score": _run_score}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    op = case["op"]
    if op == "score":
        size = 2 if case["dtype"] == "bf16" else 4
        out = case["rows"] * (8 * case["tokens"] + 4 + 8 * case["top_k"])
        return {"bytes": case["rows"] * case["vocab"] * size + out,
                "flops": 4 * case["rows"] * case["vocab"]}
    kvh, hd = case["kv_heads"], case["head_dim"]
    lens = _lens(case)
    held = 2 * kvh * (hd * ELEMENT[case["fmt"]] + (4 if case["fmt"] == "q8" else 0))
    if op == "read":
        return {"bytes": sum(lens) * (held + 8 * kvh * hd), "flops": 2 * sum(lens) * kvh * hd}
    h, counts = case["heads"], _counts(case)
    if op == "append":
        rows = sum(counts)
        return {"bytes": rows * (4 * (2 * h + 2 * kvh) * hd + 2 * held + 8 * kvh * hd),
                "flops": rows * (10 * (h + kvh) + 4 * kvh) * hd}
    # the pairing of lengths and counts goes by the seed: their means
    n = case["n"]
    rows, mean = sum(counts), sum(lens) / n
    return {"bytes": int(sum(lens) + rows) * held + 8 * rows * h * hd,
            "flops": int(4 * rows * (mean + 1) * h * hd)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def _exact_paths(parents, rows, tree):
    """For each row the rows it sees, itself last."""
    paths = []
    for t in range(rows):
        p = int(parents[t]) if tree else t - 1
        paths.append((paths[p] if p >= 0 else []) + [t])
    return paths


def _exact_values(rows, fmt):
    """What the format holds of f32 rows, in float64 (numpy)."""
    if fmt == "f16":
        return rows.astype(np.float16).astype(np.float64)
    wide = rows.astype(np.float64)
    if fmt == "f32":
        return wide
    scale = (np.abs(wide).max(-1, keepdims=True) / 127).astype(np.float32).astype(np.float64)
    return np.rint(wide / scale) * scale


def _exact_angles(case):
    d, theta, s = case["rot_dim"], case["theta"], SCALING[case["scaling"]]
    out, mag = [], 1.0
    for i in range(d // 2):
        f = math.exp(-2.0 * i / d * math.log(theta))
        if s is not None and s["kind"] == "linear":
            f /= s["factor"]
        elif s is not None and s["kind"] == "yarn":
            at = [d / (2 * math.log(theta)) * math.log(s["original"] / (2 * math.pi * b))
                  for b in (s["beta_fast"], s["beta_slow"])]
            lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), d - 1)
            w = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f = f * (1 - w) + f / s["factor"] * w
            mag = 1.0 + 0.1 * math.log(s["factor"])
        elif s is not None:
            wave = 2 * math.pi / f
            if wave > s["original"] / s["low"]:
                f /= s["factor"]
            elif wave > s["original"] / s["high"]:
                w = (s["original"] / wave - s["low"]) / (s["high"] - s["low"])
                f = w * f + (1 - w) * f / s["factor"]
        out.append(f)
    return np.array(out), mag


def _exact_append(case, x):
    n, rows, h, kvh, hd = (case[k] for k in ("n", "rows", "heads", "kv_heads", "head_dim"))
    d = case["rot_dim"]
    qkv = x["qkv"].cpu().numpy().reshape(n, rows, h + 2 * kvh, hd)
    weight = np.concatenate([np.repeat(x["q_norm"].cpu().numpy()[None], h, 0),
                             np.repeat(x["k_norm"].cpu().numpy()[None], kvh, 0)]).astype(np.float64)
    lens, counts, parents = (x[k].cpu().numpy() for k in ("lens", "counts", "parents"))
    freq, mag = _exact_angles(case)
    out = {"q": np.zeros((n, rows, h, hd)), "k": np.zeros((n, rows, kvh, hd)),
           "v": np.zeros((n, rows, kvh, hd))}
    for b in range(n):
        depth = np.array([len(p) - 1 for p in _exact_paths(parents[b], rows, case["tree"])]) \
            if case["tree"] else np.arange(rows)
        c = int(counts[b])
        y = qkv[b, :c, :h + kvh].astype(np.float64)
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + EPS) * weight
        turn = (np.exp(1j * ((lens[b] + depth[:c])[:, None] * freq)) * mag)[:, None, :]
        if case["interleaved"]:
            z = (y[..., 0:d:2] + 1j * y[..., 1:d:2]) * turn
            y[..., 0:d:2], y[..., 1:d:2] = z.real, z.imag
        else:
            z = (y[..., :d // 2] + 1j * y[..., d // 2:d]) * turn
            y[..., :d // 2], y[..., d // 2:d] = z.real, z.imag
        out["q"][b, :c] = y[:, :h]
        out["k"][b, :c] = _exact_values(y[:, h:].astype(np.float32), case["fmt"])
        out["v"][b, :c] = _exact_values(qkv[b, :c, h + kvh:], case["fmt"])
    return out


def _exact_read(case, x):
    out = {}
    for part in ("k", "v"):
        rows = x[part].cpu().numpy()
        out[part] = np.zeros(rows.shape)
        for b, c in enumerate(x["lens"].tolist()):
            out[part][b, :c] = _exact_values(rows[b, :c], case["fmt"])
    return out


def _exact_attend(case, x):
    n, rows, h, kvh, hd = (case[k] for k in ("n", "rows", "heads", "kv_heads", "head_dim"))
    g = h // kvh
    lens, counts, parents = (x[k].cpu().numpy() for k in ("lens", "counts", "parents"))
    out = torch.zeros(n, rows, h, hd, dtype=torch.float64, device="cuda")
    for b in range(n):
        length, c = int(lens[b]), int(counts[b])
        sees = np.zeros((c, length + c), bool)
        sees[:, :length] = True
        if case["tree"]:
            for t, path in enumerate(_exact_paths(parents[b], rows, True)[:c]):
                sees[t, [length + p for p in path]] = True
        else:
            sees[:, length:] = np.tri(c, dtype=bool)
        hidden = torch.from_numpy(~sees).cuda()
        for a in range(kvh):
            k, v = (torch.from_numpy(_exact_values(x[p][b, :length + c, a].cpu().numpy(),
                                                   case["fmt"])).cuda() for p in ("k", "v"))
            for head in range(a * g, a * g + g):
                z = x["q"][b, :c, head].double().matmul(k.t()) / math.sqrt(hd)
                out[b, :c, head] = torch.softmax(z.masked_fill(hidden, -math.inf), -1).matmul(v)
    return {"out": out}


def _exact_score(case, x):
    z = x["logits"].cpu().to(torch.float64)
    lse = torch.logsumexp(z, -1, keepdim=True)
    logp = z - lse
    p = torch.exp(logp)
    answer = {"logprobs": logp.gather(1, x["tokens"].cpu().long()),
              "entropy": -(p * logp).nan_to_num(0.0).sum(-1)}
    if case["top_k"]:
        order = np.argsort(-z.numpy(), axis=-1, kind="stable")[:, :case["top_k"]]
        answer["top_ids"] = torch.from_numpy(order.astype(np.int32))
        answer["top_logprobs"] = logp.gather(1, torch.from_numpy(order.copy()))
    return answer


def exact(case, seed):
    x = _inputs(case, seed)
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend,
            "score": _exact_score}[case["op"]](case, x)
