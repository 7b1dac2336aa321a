"""Contexts whose caches are in 4 bits: prompts, single rows, drafted trees, batches, the
forward without allocations and the frame step, against float64."""
import gc

import numpy as np
import pytest

import draft_ref as ref
import pages_ref as pref
import q3h
import q3o
import synth
from test_gpu_draft_forward import DIMS, HD, KVH, Model64, Setup, VOCAB, rel, rows_of

pytestmark = pytest.mark.gpu

# An element next to the border between two goes the other way where the row's f32 is an
# ulp off: a step of 1 / 7 of its 32 instead of 1 / 127 of its row, 18 times what the bar of
# int8 caches (1e-3) is for.
BAR = 18e-3
CASES = {
    "q4": dict(fmt=q3h.KV_Q4),
    "q8_weights_q4": dict(q8=True, fmt=q3h.KV_Q4),
    "pairs_of_half_q4": dict(fmt=q3h.KV_Q4, rope=dict(theta=1e4, rot_dim=64, interleaved=True)),
    "pairs_of_20_q4": dict(fmt=q3h.KV_Q4, rope=dict(theta=1e4, rot_dim=20)),
}


@pytest.fixture(autouse=True)
def four_bits(monkeypatch):
    """The float64 model's caches as 4 bits hold them."""
    monkeypatch.setattr(ref, "stored", lambda x, fmt: pref.stored(x, q3h.KV_Q4))
    yield
    gc.collect()


@pytest.mark.parametrize("case", list(CASES))
@pytest.mark.parametrize("prompt", [1, 3, 20, 90])
def test_a_tree_and_its_kept_path(device, case, prompt):
    print(f"tree {case} after {prompt}", flush=True)
    s = Setup(device, **CASES[case])
    m, c = Model64(s), s.context()
    x = rows_of(prompt, prompt)
    logits, normed = c.forward(x, head=s.head)
    want = m.forward(x)
    assert rel(normed, want[-1]) <= BAR and rel(logits, m.logits(want)[-1]) <= BAR
    for rows, seed in ((7, 1), (1, 2), (23, 3)):
        rng = np.random.default_rng(seed)
        parents = np.maximum(np.arange(rows) - rng.geometric(0.4, rows), -1).astype(np.int32)
        x = rows_of(100 + seed, rows)
        tokens = rng.integers(0, VOCAB, (rows, 2))
        got = c.forward_tree(x, parents, head=s.head, tokens=tokens, top_k=5, want_scores=True)
        want = m.forward(x, parents)
        assert c.length == len(m.cache[0])
        assert rel(got["normed"], want) <= BAR
        assert rel(got["logits"], m.logits(want)) <= BAR
        kept = ref.path(parents, int(rng.integers(rows)))[::-1]
        c.keep(kept)
        m.keep(kept)
        x = rows_of(200 + seed, 1)
        logits, normed = c.forward(x, head=s.head)
        want = m.forward(x)
        assert rel(logits, m.logits(want)[0]) <= BAR
    for layer in range(DIMS["layers"]):
        k, v = c.read_kv(layer)
        for got, part in ((k, 0), (v, 1)):
            want = np.array([row[part] for row in m.cache[layer]]).transpose(1, 0, 2)
            # an element that falls the other way is a step of its 32 off, and where the
            # step itself does (a whole number of the row's scale), each of the 32 by up to
            # one and 7 scales; the rows differ as the layers' states do
            most = np.abs(want).reshape(want.shape[:2] + (-1, 32)).max(-1, keepdims=True)
            step = np.repeat(most * 1.01 / 7, 32, -1).reshape(want.shape) + \
                np.abs(want).max(-1, keepdims=True) * (8 / 1785)
            off = np.abs(got - want)
            assert (off <= step + BAR * np.abs(want).max()).all()
            # few do
            assert (off > 1e-3 * np.abs(want).max()).mean() <= 0.02
    s.destroy(c)


@pytest.mark.parametrize("case", ["q4", "q8_weights_q4"])
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
    assert rel(got, want) <= BAR
    still = s.context()
    still.forward(x[:300], head=s.head)
    still.forward(x[300:329], head=s.head, noalloc=True)
    got, _ = still.forward(x[329:], head=s.head, noalloc=True)
    assert rel(got, want) <= BAR
    many = [s.context(n) for n in (340, 700, 500)]
    for c, n in zip(many, (329, 40, 329)):
        c.forward(x[:n], head=s.head)
    for _ in range(3):  # plain launches, then the captured ones
        lg, _ = q3h.forward_batch(many, np.stack([x[329], x[40], x[329]]), [s.head] * 3)
        assert rel(lg[0], want) <= BAR and rel(lg[2], want) <= BAR
        np.testing.assert_array_equal(lg[0], lg[2])
        for c, n in zip(many, (329, 40, 329)):
            # (what 4 bits hold may be held otherwise: a group's largest, rounded up to f32,
            # takes a step of one scale more)
            k, v = (np.stack(t) for t in zip(*[c.read_kv(i) for i in range(DIMS["layers"])]))
            c.fill_kv(k[:, :, :n], v[:, :, :n])
            again = c.read_kv(1)
            np.testing.assert_array_equal(again[0], pref.stored(k[1][:, :n], q3h.KV_Q4))
            np.testing.assert_array_equal(again[1], pref.stored(v[1][:, :n], q3h.KV_Q4))
    s.destroy(whole, one, still, *many)


def test_fill_and_read(device):
    s = Setup(device, fmt=q3h.KV_Q4)
    c = s.context(50)
    rng = np.random.default_rng(4)
    k, v = (rng.standard_normal((2, KVH, 33, HD)).astype(np.float32) for _ in range(2))
    k[0, 0, 0] = 0
    k[0, 2, 4, 32:64] *= 1e-4
    k[1, 3, 5, 7] = np.inf
    c.fill_kv(k, v)
    assert c.length == 33
    for l in range(2):
        a, b = c.read_kv(l)
        np.testing.assert_array_equal(a, pref.stored(k[l], q3h.KV_Q4))
        np.testing.assert_array_equal(b, pref.stored(v[l], q3h.KV_Q4))
    s.destroy(c)


def test_a_frame(device):
    """The frame step with both stacks' caches in 4 bits: the prefill's state is
    that of the context's forward, captured steps are the direct ones'."""
    dims = dict(synth.TALKER, layers=2)
    tl, tf = synth.stack_weights(3, "talker.model.", dims, norm_std=0.1, quantize=q3o.quantize_q8_0)
    cl, cf = synth.stack_weights(3, "talker.code_predictor.model.", dims, norm_std=0.1,
                                 quantize=q3o.quantize_q8_0)
    ts = q3h.Stack(device, dict(dims, dtype=q3h.Q8_0, kv_f16=q3h.KV_Q4, act_q8=0,
                                max_positions=256), tl, tf, q3h.Q8_0)
    cs = q3h.Stack(device, dict(dims, dtype=q3h.Q8_0, kv_f16=q3h.KV_Q4, act_q8=0,
                                max_positions=16), cl, cf, q3h.Q8_0)
    ts.add_head(q3o.quantize_q8_0(synth.talker_head(3)), q3h.Q8_0)
    for g in range(15):
        cs.add_head(q3o.quantize_q8_0(synth.cp_head(3, g)), q3h.Q8_0)
    tables = (synth.codec_embedding(3), [synth.pred_embedding(3, g) for g in range(15)],
              synth.tts_pad(3))
    prompts = [synth.prompt(3, n) for n in (12, 70)]
    frames = [q3h.Frame(ts, cs, *tables, n_streams=2, max_frames=8, max_positions=256,
                        use_graph=g) for g in (True, False)]
    for i, p in enumerate(prompts):
        frames[0].start(i, p)
    frames[1].start_batch([0, 1], prompts)
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
    for f in frames:
        f.destroy()
    c.destroy()
    ts.destroy()
    cs.destroy()


def test_quantized_activations_are_refused(device):
    layers, final = synth.stack_weights(5, "talker.model.", DIMS, quantize=q3o.quantize_q8_0)
    with pytest.raises(q3h.Q3HError) as e:
        q3h.Stack(device, dict(DIMS, dtype=q3h.Q8_0, kv_f16=q3h.KV_Q4, act_q8=1, max_positions=64),
                  layers, final, q3h.Q8_0)
    assert e.value.code == q3h.E_ARG
