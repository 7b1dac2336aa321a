"""Drafted trees and rows over int8 caches on contexts, where the attention's
groups are cut into shares that leave parts (contexts of more than a few hundred
positions), and what other calls on a context do to a pending tree."""
import gc

import numpy as np
import pytest
import torch

import draft_ref as ref
import q3h
from test_gpu_draft_forward import (CASES, DIMS, HD, HEADS, KVH, Model64, Setup, bar, rel,
                                    rows_of)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_handles_left():
    yield
    gc.collect()


@pytest.mark.parametrize("fmt", [q3h.KV_F32, q3h.KV_F16])
def test_a_measured_attention_drops_the_tree(device, fmt):
    """q3h_context_time_attention writes position len, where the tree's first row
    waits: nothing of the tree can be kept after it."""
    s = Setup(device, fmt=fmt)
    c = s.context(60)
    x = rows_of(1, 4)
    c.forward(x[:2])
    c.forward_tree(x, [-1, 0, 1, 0])
    c.time_attention(iters=1)
    with pytest.raises(q3h.Q3HError) as e:
        c.keep([0, 1])
    assert e.value.code == q3h.E_STATE and c.length == 2
    c.forward_tree(x, [-1, 0, 1, 0])
    c.keep([0, 1])
    assert c.length == 4
    s.destroy(c)


# ---------------------------------------------------------------------------
# long contexts


def cut(device, s, rows, positions):
    """Whether the attention of rows over so many positions leaves parts."""
    c = q3h.Cache(device, 1, KVH, HD, positions, s.fmt)
    need = c.attend_workspace(1, rows, HEADS, positions - rows)
    c.destroy()
    return need > 0


def filled(s, c, m, n, seed=3):
    """n random positions in the context c and in the models m."""
    rng = np.random.default_rng(seed)
    k, v = (rng.standard_normal((DIMS["layers"], KVH, n, HD)).astype(np.float32)
            for _ in range(2))
    c.fill_kv(k, v)
    for model in m:
        for l in range(DIMS["layers"]):
            a, b = (ref.stored(t[l], s.fmt).astype(np.float64) for t in (k, v))
            model.cache[l] = [(a[:, p], b[:, p]) for p in range(n)]


def drafted_tree(rows, seed):
    rng = np.random.default_rng(seed)
    return np.maximum(np.arange(rows) - rng.geometric(0.4, rows), -1).astype(np.int32)


LONG = 2304
LONG_CASES = ["f32", "f16", "int8", "q8_weights_int8", "yarn"]


@pytest.mark.parametrize("case", LONG_CASES)
def test_trees_and_rows_of_long_contexts(device, case):
    """A tree of each size of group, a path of it kept, then single rows: direct,
    replayed, of a batch, without allocations, over 1500 positions and more,
    against float64."""
    print(f"long {case}", flush=True)
    s = Setup(device, max_positions=LONG, **CASES[case])
    own = CASES[case].get("fmt") == q3h.KV_Q8 or "rope" in CASES[case]
    m, c = Model64(s), s.context(LONG)
    filled(s, c, [m], 1500)
    for rows, seed in ((7, 1), (23, 2), (64, 3), (1, 4)):
        assert cut(device, s, rows, c.length + rows)
        parents, x = drafted_tree(rows, seed), rows_of(100 + seed, rows)
        got = c.forward_tree(x, parents, head=s.head)
        want = m.forward(x, parents)
        assert rel(got["normed"], want) <= bar(case)
        assert rel(got["logits"], m.logits(want)) <= bar(case)
        kept = ref.path(parents, rows - 1)[::-1]
        c.keep(kept)
        m.keep(kept)
        assert c.length == len(m.cache[0])
        for i, noalloc in enumerate((False, False, True)):
            assert not own or cut(device, s, 1, c.length + 1)
            x = rows_of(200 + 10 * seed + i, 1)
            logits, normed = c.forward(x, head=s.head, noalloc=noalloc)
            want = m.forward(x)
            assert rel(normed, want[0]) <= bar(case)
            assert rel(logits, m.logits(want)[0]) <= bar(case)
    x = rows_of(300, 20)
    logits, _ = c.forward(x, head=s.head)  # several rows
    want = m.forward(x)
    assert rel(logits, m.logits(want)[-1]) <= bar(case)
    # a batch whose first context is short: plain launches, then the captured ones
    d, n = s.context(LONG), Model64(s)
    filled(s, d, [n], 30)
    for i in range(3):
        x = rows_of(400 + i, 2)
        lg, _ = q3h.forward_batch([d, c], x, [s.head] * 2)
        assert rel(lg[0], n.logits(n.forward(x[:1]))[0]) <= bar(case)
        assert rel(lg[1], m.logits(m.forward(x[1:]))[0]) <= bar(case)
    s.destroy(c, d)


@pytest.mark.parametrize("case", ["int8", "yarn"])
@pytest.mark.parametrize("positions", [700, 1500, 4000])
def test_forwards_without_allocations_at_any_length(device, case, positions):
    """Up to 64 rows in the device's array, whose room for the attention's parts
    is less than they ask for: fewer parts, the results of q3h_forward_embeds but
    for the order of sums."""
    print(f"noalloc {case} {positions}", flush=True)
    s = Setup(device, max_positions=4096, **CASES[case])
    a, b, m = s.context(4096), s.context(4096), Model64(s)
    for rows in (64, 48, 30, 17, 2):
        for c in (a, b):
            filled(s, c, [m] if c is a else [], positions)
        assert rows == 2 or cut(device, s, rows, positions + rows)
        x = rows_of(rows, rows)
        la, na = a.forward(x, head=s.head, noalloc=True)
        lb, nb = b.forward(x, head=s.head)
        assert rel(la, lb) <= bar(case) and rel(na, nb) <= bar(case)
        if rows in (64, 2):
            want = m.forward(x)
            assert rel(la, m.logits(want)[-1]) <= bar(case)
    s.destroy(a, b)


@pytest.mark.parametrize("case", ["f32", "int8"])
def test_trees_of_a_growing_context_allocate_once(device, case):
    """The parts of a tree's attention: room for those of the context's last
    position from the first tree that leaves any."""
    print(f"growing {case}", flush=True)
    s = Setup(device, max_positions=4096, **CASES[case])
    c = s.context(4096)
    x, parents = rows_of(5, 64), drafted_tree(64, 5)
    # (the other buffers at their largest: 64 rows, a single row's splits at the end)
    c.forward_tree(x, parents, head=s.head)
    filled(s, c, [], 4095)
    c.forward(x[:1], head=s.head)
    free = []
    for n in (700, 900, 1300, 2100, 3000, 4000):
        filled(s, c, [], n)
        c.forward_tree(x, parents, head=s.head)
        c.keep([0])
        c.forward(x[:1], head=s.head)
        torch.cuda.synchronize()
        free.append(torch.cuda.mem_get_info()[0])
    assert len(set(free)) == 1, free
    s.destroy(c)
