"""Drafted trees, int8 caches, other rotary positions and scored rows through
the layers of a stack (q3h_forward_tree, q3h_context_keep, q3h_forward_score,
q3h_stack_set_rope) against float64."""
import ctypes
import gc

import numpy as np
import pytest

import draft_ref as ref
import q3h
import q3o
import synth

pytestmark = pytest.mark.gpu

DIMS = dict(synth.TALKER, layers=2, intermediate=2048)
H, HEADS, KVH, HD = DIMS["hidden"], DIMS["heads"], DIMS["kv_heads"], DIMS["head_dim"]
VOCAB = 1040
# the bars of the stacks' other forwards: f32 products, Q8_0 weights (exact
# here: the reference takes the dequantized ones); an int8 cache's byte next to
# a half may go the other way, one step of 1 / 127 in one of its 128 elements
F32_BAR, Q8_BAR = 1e-4, 1e-3


@pytest.fixture(autouse=True)
def no_handles_left():
    yield
    gc.collect()


class Setup:
    """A stack and its weights in float64."""

    def __init__(self, device, fmt=q3h.KV_F32, q8=False, act_q8=0, rope=None, seed=5,
                 max_positions=700):
        quant = q3o.quantize_q8_0 if q8 else None
        self.fmt, self.rope = fmt, rope
        plain, self.final = synth.stack_weights(seed, "talker.model.", DIMS, norm_std=0.1)
        layers, _ = synth.stack_weights(seed, "talker.model.", DIMS, norm_std=0.1, quantize=quant)
        head = synth.normal(seed, "head", (VOCAB, H))
        src = q3h.Q8_0 if q8 else q3h.F32
        self.stack = q3h.Stack(device, dict(DIMS, dtype=src, kv_f16=fmt, act_q8=act_q8,
                                            max_positions=max_positions), layers, self.final, src)
        if rope is not None:
            self.stack.set_rope(**rope)
        self.head = self.stack.add_head(quant(head) if q8 else head, src)

        def wide(w):
            return dequantized(quant(w)) if q8 else w.astype(np.float64)
        self.layers = [{k: wide(v) if v.ndim == 2 else v.astype(np.float64)
                        for k, v in L.items()} for L in plain]
        self.head64 = wide(head)

    def context(self, n=700):
        return q3h.Context(self.stack, n)

    def destroy(self, *contexts):
        for c in contexts:
            c.destroy()
        self.stack.destroy()


def dequantized(blocks):
    b = blocks.reshape(blocks.shape[0], -1, 34)
    d = np.ascontiguousarray(b[:, :, :2]).view(np.float16).astype(np.float64)
    return (b[:, :, 2:].view(np.int8) * d).reshape(blocks.shape[0], -1)


class Model64:
    """The stack's forward in float64, its cache as the format holds it."""

    def __init__(self, s):
        self.s = s
        self.cache = [[] for _ in s.layers]  # (k, v) [kvh][hd] of each position
        if s.rope is None:
            # the stack's own table: the angle an f32 product
            self.f32 = (1.0 / DIMS["rope_theta"] ** (2 * np.arange(HD // 2) / HD)).astype(np.float32)

    def turn(self, x, pos):
        r = self.s.rope
        if r is None:
            angle = (np.float32(pos) * self.f32).astype(np.float64)
            return ref.turned(x, 1, HD, False, angle, 1.0)
        rot = r.get("rot_dim") or HD
        f, mag = ref.frequencies(rot, r["theta"], r.get("scaling"))
        return ref.turned(x, pos, rot, r.get("interleaved", False), f, mag)

    def forward(self, x, parents=None):
        """The rows' normed states; the cache grows by the rows of a chain, by
        none of a tree (self.drafted keeps them)."""
        base = len(self.cache[0])
        h = x.astype(np.float64)
        rows = len(h)
        paths = [ref.path(parents, t) for t in range(rows)]
        drafted = []
        for L, held in zip(self.s.layers, self.cache):
            n = ref.normed(h, L["input_norm"], DIMS["rms_eps"])
            q = (n @ L["wq"].T).reshape(rows, HEADS, HD)
            k = (n @ L["wk"].T).reshape(rows, KVH, HD)
            v = (n @ L["wv"].T).reshape(rows, KVH, HD)
            q = ref.normed(q, L["q_norm"], DIMS["rms_eps"])
            k = ref.normed(k, L["k_norm"], DIMS["rms_eps"])
            new = []
            for t in range(rows):
                pos = base + len(paths[t]) - 1
                q[t] = self.turn(q[t], pos)
                kt = ref.stored(self.turn(k[t], pos).astype(np.float32), self.s.fmt)
                new.append((kt.astype(np.float64),
                            ref.stored(v[t].astype(np.float32), self.s.fmt).astype(np.float64)))
            o = np.zeros((rows, HEADS, HD))
            for t in range(rows):
                seen = held + [new[r] for r in sorted(paths[t])]
                kk, vv = np.array([a for a, _ in seen]), np.array([b for _, b in seen])
                for a in range(HEADS):
                    s = kk[:, a // 2] @ q[t, a] / np.sqrt(HD)
                    p = np.exp(s - s.max())
                    o[t, a] = p / p.sum() @ vv[:, a // 2]
            h = h + o.reshape(rows, -1) @ L["wo"].T
            n = ref.normed(h, L["post_norm"], DIMS["rms_eps"])
            g = n @ L["wgate"].T
            h = h + (g / (1 + np.exp(-g)) * (n @ L["wup"].T)) @ L["wdown"].T
            drafted.append(new)
        self.drafted = drafted
        if parents is None:
            self.keep(range(rows))
        return ref.normed(h, self.s.final.astype(np.float64), DIMS["rms_eps"])

    def keep(self, rows):
        for held, new in zip(self.cache, self.drafted):
            held += [new[r] for r in rows]

    def logits(self, normed):
        return normed @ self.s.head64.T


def rel(a, b):
    return float(np.abs(a - b).max() / np.abs(b).max())


def rows_of(seed, n):
    return np.random.default_rng(seed).standard_normal((n, H)).astype(np.float32)


CASES = {
    "f32": dict(),
    "f16": dict(fmt=q3h.KV_F16),
    "int8": dict(fmt=q3h.KV_Q8),
    "q8_weights": dict(q8=True),
    "q8_weights_int8": dict(q8=True, fmt=q3h.KV_Q8),
    "yarn": dict(rope=dict(theta=1e4, scaling=dict(kind="yarn", factor=4.0, original=64))),
    "pairs_of_half_int8": dict(fmt=q3h.KV_Q8, rope=dict(theta=1e4, rot_dim=64, interleaved=True)),
    "bands_f16": dict(fmt=q3h.KV_F16, q8=True,
                      rope=dict(theta=1e6, scaling=dict(kind="bands", factor=8.0, original=128))),
}


def bar(case):
    c = CASES[case]
    # (an f16 cache rounds on the way: a tie may fall the other way, 2^-11)
    return F32_BAR if c.get("fmt", 0) == q3h.KV_F32 else Q8_BAR


@pytest.mark.parametrize("case", list(CASES))
@pytest.mark.parametrize("prompt", [1, 3, 20, 90])
def test_a_tree_and_its_kept_path(device, case, prompt):
    """A prompt (each way the products take rows), a drafted tree, a path of it
    kept, the next token, and the caches read back."""
    print(f"tree {case} after {prompt}", flush=True)
    s = Setup(device, **CASES[case])
    m, c = Model64(s), s.context()
    x = rows_of(prompt, prompt)
    logits, normed = c.forward(x, head=s.head)
    want = m.forward(x)
    assert rel(normed, want[-1]) <= bar(case) and rel(logits, m.logits(want)[-1]) <= bar(case)
    for rows, seed in ((7, 1), (1, 2), (23, 3)):
        rng = np.random.default_rng(seed)
        parents = np.maximum(np.arange(rows) - rng.geometric(0.4, rows), -1).astype(np.int32)
        x = rows_of(100 + seed, rows)
        tokens = rng.integers(0, VOCAB, (rows, 2))
        got = c.forward_tree(x, parents, head=s.head, tokens=tokens, top_k=5, want_scores=True)
        want = m.forward(x, parents)
        assert c.length == len(m.cache[0])
        assert rel(got["normed"], want) <= bar(case)
        assert rel(got["logits"], m.logits(want)) <= bar(case)
        lp, ent, ids, top = ref.scores(got["logits"], tokens, 5)
        np.testing.assert_array_equal(got["top_ids"], ids)
        # logits of a few units, sums of 1040 terms: as the scores' own test
        for name, w in (("logprobs", lp), ("entropy", ent), ("top_logprobs", top)):
            np.testing.assert_allclose(got[name], w, rtol=0, atol=2e-5)
        kept = ref.path(parents, int(rng.integers(rows)))[::-1]
        c.keep(kept)
        m.keep(kept)
        assert c.length == len(m.cache[0])
        x = rows_of(200 + seed, 1)
        logits, normed = c.forward(x, head=s.head)
        want = m.forward(x)
        assert rel(logits, m.logits(want)[0]) <= bar(case)
    for layer in range(DIMS["layers"]):
        k, v = c.read_kv(layer)
        for got, part in ((k, 0), (v, 1)):
            want = np.array([row[part] for row in m.cache[layer]]).transpose(1, 0, 2)
            # a value that falls the other way is one step of its row off
            step = np.abs(want).max(-1, keepdims=True) * (1.02 / 127 if s.fmt == q3h.KV_Q8
                                                          else 2.0 ** -10)
            assert (np.abs(got - want) <= step + 1e-4 * np.abs(want).max()).all()
    s.destroy(c)


@pytest.mark.parametrize("case", ["f32", "int8", "q8_weights", "act_q8", "act_q8_f16"])
@pytest.mark.parametrize("rows", [1, 4, 40, 100])
def test_scored_rows(device, case, rows):
    """forward_score: the state of forward(), the scores of every row's logits."""
    kw = dict(q8=True, act_q8=1, fmt=q3h.KV_F16 if case.endswith("f16") else q3h.KV_F32) \
        if case.startswith("act_q8") else CASES[case]
    s = Setup(device, **kw)
    a, b = s.context(201), s.context(201)
    x = rows_of(7, rows)
    tokens = np.random.default_rng(8).integers(0, VOCAB, (rows, 3))
    tokens[0, 0] = -1
    for _ in range(2):
        got = a.forward_score(x, s.head, tokens=tokens, top_k=3, want_logits=True, want_normed=True)
        logits, normed = b.forward(x, head=s.head)
        assert a.length == b.length
        # the same layers over the same rows; the head's product takes them all at once
        np.testing.assert_array_equal(got["normed"][-1], normed)
        assert rel(got["logits"][-1], logits) <= F32_BAR
        lp, ent, ids, top = ref.scores(got["logits"], tokens, 3)
        np.testing.assert_array_equal(got["top_ids"], ids)
        assert np.isnan(got["logprobs"][0, 0]) and np.isnan(lp[0, 0])
        for name, w in (("logprobs", lp), ("entropy", ent), ("top_logprobs", top)):
            np.testing.assert_allclose(got[name], w, rtol=0, atol=2e-5)
    none = a.forward_score(x[:1], s.head)
    assert none["logprobs"].shape == (1, 0) and np.isfinite(none["entropy"]).all()
    s.destroy(a, b)


@pytest.mark.parametrize("case", ["int8", "q8_weights_int8", "yarn"])
def test_every_forward_of_a_stack(device, case):
    """One row after another past each cover of the captured launches, several
    contexts at once, and the forward without allocations: as one prompt."""
    s = Setup(device, **CASES[case])
    x = rows_of(11, 330)
    whole = s.context()
    want, _ = whole.forward(x, head=s.head)
    one = s.context()
    one.forward(x[:60], head=s.head)
    for i in range(60, 330):
        got, _ = one.forward(x[i:i + 1], head=s.head)
    assert rel(got, want) <= bar(case)
    still = s.context()
    still.forward(x[:300], head=s.head)
    still.forward(x[300:329], head=s.head, noalloc=True)
    got, _ = still.forward(x[329:], head=s.head, noalloc=True)
    assert rel(got, want) <= bar(case)
    many = [s.context(n) for n in (340, 700, 500)]
    for c, n in zip(many, (329, 40, 329)):
        c.forward(x[:n], head=s.head)
    for _ in range(3):  # plain launches, then the captured ones
        lg, _ = q3h.forward_batch(many, np.stack([x[329], x[40], x[329]]), [s.head] * 3)
        assert rel(lg[0], want) <= bar(case) and rel(lg[2], want) <= bar(case)
        np.testing.assert_array_equal(lg[0], lg[2])
        for c, n in zip(many, (329, 40, 329)):
            k, v = (np.stack(t) for t in zip(*[c.read_kv(i) for i in range(DIMS["layers"])]))
            c.fill_kv(k[:, :, :n], v[:, :, :n])
    s.destroy(whole, one, still, *many)


def test_fill_and_read_an_int8_cache(device):
    s = Setup(device, fmt=q3h.KV_Q8)
    c = s.context(50)
    rng = np.random.default_rng(4)
    k, v = (rng.standard_normal((2, KVH, 33, HD)).astype(np.float32) for _ in range(2))
    k[0, 0, 0] = 0
    k[1, 3, 5, 7] = np.inf
    c.fill_kv(k, v)
    assert c.length == 33
    for l in range(2):
        a, b = c.read_kv(l)
        np.testing.assert_array_equal(a, ref.stored(k[l], 2))
        np.testing.assert_array_equal(b, ref.stored(v[l], 2))
    s.destroy(c)


def test_a_frame_over_int8_caches(device):
    """The frame step with both stacks' caches in int8: the prefill's state is
    that of the context's forward, captured steps are the direct ones', streams
    started together are those started one by one."""
    rng = np.random.default_rng(6)
    dims = dict(synth.TALKER, layers=2)
    tl, tf = synth.stack_weights(3, "talker.model.", dims, norm_std=0.1, quantize=q3o.quantize_q8_0)
    cl, cf = synth.stack_weights(3, "talker.code_predictor.model.", dims, norm_std=0.1,
                                 quantize=q3o.quantize_q8_0)
    ts = q3h.Stack(device, dict(dims, dtype=q3h.Q8_0, kv_f16=q3h.KV_Q8, act_q8=0,
                                max_positions=256), tl, tf, q3h.Q8_0)
    cs = q3h.Stack(device, dict(dims, dtype=q3h.Q8_0, kv_f16=q3h.KV_Q8, act_q8=0,
                                max_positions=16), cl, cf, q3h.Q8_0)
    ts.add_head(q3o.quantize_q8_0(synth.talker_head(3)), q3h.Q8_0)
    for g in range(15):
        cs.add_head(q3o.quantize_q8_0(synth.cp_head(3, g)), q3h.Q8_0)
    tables = (synth.codec_embedding(3), [synth.pred_embedding(3, g) for g in range(15)],
              synth.tts_pad(3))
    prompts = [synth.prompt(3, n) for n in (12, 70, 100)]
    frames = [q3h.Frame(ts, cs, *tables, n_streams=3, max_frames=8, max_positions=256,
                        use_graph=g) for g in (True, False)]
    for i, p in enumerate(prompts):
        frames[0].start(i, p)
    frames[1].start_batch([0, 1, 2], prompts)
    c = q3h.Context(ts, 256)
    for i, p in enumerate(prompts):
        c.reset()
        logits, _ = c.forward(p, head=0)
        lg, _ = frames[0].state(i)
        np.testing.assert_array_equal(lg, logits)
        np.testing.assert_array_equal(frames[1].state(i)[0], lg)
    for _ in range(4):
        a, alive = frames[0].step()
        b, _ = frames[1].step()
        np.testing.assert_array_equal(a, b)
        assert alive.all() and (a >= 0).all()
    # a lone stream: none of the fused code-predictor launches, the same codes
    one = q3h.Frame(ts, cs, *tables, n_streams=1, max_frames=8, max_positions=256)
    one.start(0, prompts[1])
    one_codes = one.step()[0]
    assert one_codes.shape == (1, 16) and (one_codes >= 0).all()
    for f in frames + [one]:
        f.destroy()
    c.destroy()
    ts.destroy()
    cs.destroy()


def test_refusals(device):
    s = Setup(device)
    c = s.context(60)
    x = rows_of(1, 4)
    c.forward(x[:2])

    def code(f, *a, **k):
        with pytest.raises(q3h.Q3HError) as e:
            f(*a, **k)
        return e.value.code

    assert code(c.keep, [0]) == q3h.E_STATE
    assert code(c.forward_tree, x, [-1, 1, 0, 0]) == q3h.E_ARG
    assert code(c.forward_tree, x, [-2, 0, 0, 0]) == q3h.E_ARG
    assert code(c.forward_tree, x, [-1, 0, 0, 0], head=5) == q3h.E_ARG
    assert code(c.forward_tree, x, [-1, 0, 0, 0], want_scores=True) == q3h.E_ARG  # no head
    assert code(c.forward_tree, rows_of(1, 65)[:65], [-1] * 65) == q3h.E_CAPACITY
    assert code(c.forward_tree, rows_of(1, 60), [-1] * 60) == q3h.E_CAPACITY
    assert code(c.forward_score, x, -1) == q3h.E_ARG
    assert code(c.forward_score, x, s.head, top_k=65) == q3h.E_ARG
    assert c.length == 2
    c.forward_tree(x, [-1, 0, 1, 0])
    for bad in ([1], [0, 2], [0, 1, 3], [4], [0, 0]):
        assert code(c.keep, bad) == q3h.E_ARG
    c.keep([0, 1])
    assert c.length == 4
    assert code(c.keep, [0]) == q3h.E_STATE  # kept once
    c.forward_tree(x, [-1, 0, 1, 0])
    c.keep([])
    assert c.length == 4
    for write in (lambda: c.forward(x[:1]), lambda: c.forward(x[:1], noalloc=True),
                  lambda: q3h.forward_batch([c], x[:1]), lambda: c.forward_score(x[:1], s.head),
                  lambda: c.forward_probe(x[:1]), c.reset):
        c.forward_tree(x, [-1, 0, 1, 0])
        write()
        assert code(c.keep, [0]) == q3h.E_STATE
    assert code(s.stack.set_rope, 1e4) == q3h.E_STATE  # contexts use it
    c.destroy()
    assert code(s.stack.set_rope, 1e4, rot_dim=3) == q3h.E_ARG
    cfg = q3h.RopeConfig(HD, HD, 0, 699, 1e4)
    assert q3h.lib().q3h_stack_set_rope(s.stack.h, ctypes.byref(cfg)) == q3h.E_ARG
    s.stack.set_rope(1e4)
    s.stack.set_rope(1e5)  # again before the first context
    t = s.context(60)
    assert code(t.time_attention) == q3h.E_ARG
    s.destroy(t)
    a = Setup(device, q8=True, act_q8=1)
    d = a.context(60)
    assert code(d.forward_tree, x, [-1, 0, 0, 0]) == q3h.E_ARG
    d.destroy()
    assert code(a.stack.set_rope, 1e4) == q3h.E_ARG
    a.destroy()
    layers, final = synth.stack_weights(5, "talker.model.", DIMS, quantize=q3o.quantize_q8_0)
    for kv, act in ((3, 0), (-1, 0), (2, 1)):
        assert code(q3h.Stack, device, dict(DIMS, dtype=q3h.Q8_0, kv_f16=kv, act_q8=act,
                                            max_positions=64), layers, final,
                    q3h.Q8_0) == q3h.E_ARG


def test_arrays_that_do_not_fit_are_refused(device):
    """Before a pointer to them is handed on."""
    s = Setup(device)
    c = s.context(60)
    x = rows_of(1, 4)
    for call in (lambda: c.forward_tree(x, [-1, 0, 0]),
                 lambda: c.forward_tree(x, [[-1, 0, 0, 0]]),
                 lambda: c.forward_tree(x[:, :-1], [-1, 0, 0, 0]),
                 lambda: c.forward_tree(x, [-1, 0, 0, 0], s.head, tokens=[[1, 2, 3, 4]] * 2,
                                        want_scores=True),
                 lambda: c.forward_score(x[0], s.head),
                 lambda: c.forward_score(x, s.head, tokens=[1, 2])):
        with pytest.raises(q3h.Q3HError) as e:
            call()
        assert e.value.code == q3h.E_ARG
    assert c.length == 0
    got = c.forward_score(x, s.head, tokens=[1, 2, 3, 4])
    assert got["logprobs"].shape == (4, 1) and c.length == 4
    c.destroy()
    s.destroy()
