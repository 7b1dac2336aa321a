"""Attention over 4 bits whose even shares go from one sequence's heads to the next: up to 16
query rows of a kv head over more positions than a call that is not cut, with sequences
among them that have no rows, bad lengths, no pages, broken paths, NaN and infinities in
seen and in unseen rows, and values so small that a wave goes over its positions again."""
import numpy as np
import pytest
import torch

import draft_ref as ref
import pages_ref as pref
import q3h
from test_gpu_draft import dev_f, dev_i, host, random_tree
from test_gpu_pages import a_cache, fill

pytestmark = pytest.mark.gpu

N = q3h.KV_Q4
KINDS = ["good", "no rows", "below 0", "too long", "no room", "broken", "seen nan", "unseen nan",
         "small", "unseen inf"]

# (sequences, heads, kv heads, elements of a head, rows, tree): up to 8 query rows of a kv head
# and up to 16, fewer sequences than a wave has lanes, and more
CASES = [
    (11, 4, 2, 64, 4, True),
    (11, 8, 2, 128, 3, False),
    (11, 3, 3, 128, 1, False),
    (11, 4, 1, 64, 4, True),
    (75, 4, 2, 64, 4, True),
    (75, 6, 2, 128, 5, True),
    (140, 2, 2, 64, 1, False),
    (70, 16, 1, 64, 1, False),
]


def kinds_of(rng, n):
    """Every kind once, the others half of them good ones, in any order."""
    more = np.where(rng.random(max(0, n - len(KINDS))) < 0.5, 0,
                    rng.integers(0, len(KINDS), max(0, n - len(KINDS))))
    return [KINDS[i] for i in rng.permutation(np.concatenate([np.arange(len(KINDS)), more]))]


@pytest.mark.parametrize("page", [0, 32, 256])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_sequences_of_any_kind_share_a_call(device, case, page):
    n, heads, kvh, hd, rows, tree = CASES[case]
    print(f"{n} sequences, heads {heads} over {kvh} of {hd}, {rows} rows, tree {tree}, page {page}",
          flush=True)
    rng = np.random.default_rng(300 + case)
    kinds = kinds_of(rng, n)
    max_len, g = 1200, heads // kvh
    P = max_len + rows + 20
    lens = np.where(rng.random(n) < 0.7, rng.integers(1, max_len + 1, n), rng.integers(1, 60, n))
    lens[kinds.index("good")] = max_len
    counts = rng.integers(1, rows + 1, n)
    k = rng.standard_normal((n, P, kvh, hd)).astype(np.float32)
    v = rng.standard_normal((n, P, kvh, hd)).astype(np.float32)
    q = rng.standard_normal((n, rows, heads, hd)).astype(np.float32)
    parents = random_tree(rng, n, rows) if tree else None
    nan = np.zeros((n, rows, heads), bool)  # what has to be NaN
    held = lens + counts
    for b, kind in enumerate(kinds):
        if kind == "no rows":
            counts[b] = 0
        elif kind == "below 0":
            lens[b], nan[b] = -1 - b, True
        elif kind == "too long":
            lens[b], held[b], nan[b] = max_len + 3, P, True
        elif kind == "no room":  # behind the pages, or the cache's last position
            lens[b], held[b], nan[b] = (lens[b] if page else P), 0, True
        elif kind == "broken" and tree:
            counts[b] = rows
            parents[b, rows - 2] = rows - 1
            parents[b, rows - 1] = rows - 2 if b % 2 else -1
            held[b] = lens[b] + rows
            nan[b, rows - 2] = True
            nan[b, rows - 1] = b % 2 == 1
        elif kind == "seen nan":  # of one kv head
            at = rng.integers(0, lens[b])
            (k if b % 2 else v)[b, at, 0, 5] = np.nan if b % 3 else np.inf
            nan[b, :, :g] = True
        elif kind in ("unseen nan", "unseen inf"):
            bad = np.nan if kind == "unseen nan" else -np.inf
            if tree:  # a sibling that no row continues
                counts[b] = rows
                held[b] = lens[b] + rows
                parents[b, rows - 1] = parents[b, rows - 2] = -1
                k[b, lens[b] + rows - 2], v[b, lens[b] + rows - 2] = bad, bad
                nan[b, rows - 2] = True
            k[b, lens[b] + counts[b]:, :, 3] = bad  # behind the rows
            v[b, lens[b] + counts[b]:, :, ::2] = bad
        elif kind == "small":
            v[b] *= np.float32(2.0 ** -80)
    held = np.minimum(np.maximum(held, 0), P)
    if page == 0:
        held[:] = P
    elif page == 256:  # (to the end of the last page)
        held = np.minimum(P, -(-held // page) * page)
    cache = a_cache(device, n, kvh, hd, P, N, page, held, rng)
    fill(cache, k, v, held)
    args = dict(counts=dev_i(counts), parents=None if parents is None else dev_i(parents))
    out = torch.full((n, rows, heads, hd), 7.0, device="cuda")
    cache.attend(dev_f(q), dev_i(lens), max_len, out=out, **args)
    got = host(out)
    stored = [pref.stored(x, N).astype(np.float64) for x in (k, v)]
    checked = 0
    for b, kind in enumerate(kinds):
        assert (got[b, counts[b]:] == 7).all(), (b, kind)
        assert np.isnan(got[b, :counts[b]][nan[b, :counts[b]]]).all(), (b, kind)
        live = ~nan[b, :counts[b]]
        if not live.any():
            continue
        clean = [np.nan_to_num(x[b:b + 1], nan=0, posinf=0, neginf=0) for x in stored]
        sound = None
        if tree:
            sound = np.minimum(parents[b:b + 1], np.arange(rows) - 1)
        want, bound = ref.attention(q[b:b + 1].astype(np.float64), *clean, lens[b:b + 1],
                                    counts[b:b + 1], sound, hd ** -0.5)
        d = np.abs(got[b, :counts[b]] - want[0, :counts[b]])
        assert (d <= bound[0, :counts[b]])[live].all(), (b, kind, (d / bound[0, :counts[b]])[live].max())
        checked += 1
    print(f"{checked} sequences checked", flush=True)
    assert checked >= len(KINDS) // 2
    # the same bits again, with what the call before left in the workspace
    space = torch.full((cache.attend_workspace(n, rows, heads, max_len),), 255, dtype=torch.uint8,
                       device="cuda")
    for _ in range(2):
        again = torch.full((n, rows, heads, hd), 7.0, device="cuda")
        cache.attend(dev_f(q), dev_i(lens), max_len, out=again, workspace=space, **args)
        np.testing.assert_array_equal(host(again), got)


@pytest.mark.parametrize("n", [3, 80])
def test_no_sequence_has_rows(device, n):
    """All counts 0: there are no shares, and nothing is written."""
    cache = q3h.Cache(device, n, 2, 64, 2000, N)
    q = torch.zeros((n, 2, 4, 64), device="cuda")
    out = torch.full_like(q, 7.0)
    lens = np.full(n, 1500)
    lens[0] = -1
    cache.attend(q, dev_i(lens), 1900, out=out, counts=dev_i([0] * n))
    assert bool((out == 7).all())
    assert cache.attend_workspace(n, 2, 4, 1900) > 0


def test_captured_shares_follow_lengths_on_the_device(device):
    """A captured call over lengths and counts that change between its replays, none at all
    among them, with other work between, against the same call made eagerly."""
    rng = np.random.default_rng(7)
    n, rows, heads, kvh, hd, P = 20, 2, 8, 4, 64, 2000
    cache = q3h.Cache(device, n, kvh, hd, P, N, pages=n * 63, page_positions=32)
    cache.reserve(dev_i([0] * n), P)
    x = rng.standard_normal((n, P, kvh, hd)).astype(np.float32)
    fill(cache, x, x[::-1].copy(), [P] * n)
    q = dev_f(rng.standard_normal((n, rows, heads, hd)))
    lens, counts = dev_i([100] * n), dev_i([rows] * n)
    spaces = [torch.zeros(cache.attend_workspace(n, rows, heads, P - rows), dtype=torch.uint8,
                          device="cuda") for _ in range(2)]
    outs = [torch.zeros((n, rows, heads, hd), device="cuda") for _ in range(2)]

    def call(i):
        cache.attend(q, lens, P - rows, out=outs[i], counts=counts, workspace=spaces[i])

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        call(0)
        with torch.cuda.graph(graph, stream=side):
            call(0)
    torch.cuda.synchronize()
    for turn in range(8):
        some = rng.integers(0, rows + 1, n) if turn != 3 else np.zeros(n, int)
        at = rng.integers(0, P - rows + 1, n)
        if turn % 2:
            at[rng.integers(0, n, 3)] = [-1, P, 0]
        lens.copy_(dev_i(at))
        counts.copy_(dev_i(some))
        for out in outs:
            out.fill_(turn)
        call(1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(host(outs[0]), host(outs[1]))
        for b in range(n):
            assert (host(outs[0])[b, some[b]:] == turn).all()
            bad = not 0 <= at[b] <= P - rows
            assert bool(np.isnan(host(outs[0])[b, :some[b]]).all()) == bad or some[b] == 0
