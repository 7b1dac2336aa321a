"""Caches in 4 bits, caches in pages and rotary positions of several axes on the
device against float64 and lists, through the binding's tensors."""
import gc

import numpy as np
import pytest
import torch

import draft_ref as ref
import pages_ref as pref
import q3h
from test_gpu_draft import ROPES, dev_f, dev_i, host, random_tree

pytestmark = pytest.mark.gpu

F, H, Q, N = q3h.KV_F32, q3h.KV_F16, q3h.KV_Q8, q3h.KV_Q4
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def no_handles_left():
    """Handles that a refusal's traceback still holds go before the device does."""
    yield
    gc.collect()


def paged(device, n, kvh, hd, positions, fmt, page, layers=1, spare=3):
    """A cache in pages for n sequences of all positions and a few pages more."""
    return q3h.Cache(device, n, kvh, hd, positions, fmt, layers=layers, page_positions=page,
                     pages=n * -(-positions // page) + spare)


def scatter(cache, held, page, rng):
    """Pages for held[b] positions, the sequences' pages in any order."""
    n, held = len(held), np.asarray(held)
    most = -(-int(held.max(initial=0)) // page)
    for at in range(1, most + 1):
        for b in rng.permutation(n):
            counts = np.zeros(n, int)
            counts[b] = min(held[b], at * page)
            cache.reserve(dev_i(np.zeros(n)), max(1, int(held.max())), counts=dev_i(counts))


def fill(cache, k, v, held, layer=0):
    if k.shape[1]:
        cache.append(dev_f(k), dev_f(v), dev_i([0] * k.shape[0]), counts=dev_i(held), layer=layer)


def a_cache(device, n, kvh, hd, positions, fmt, page, held, rng, layers=1):
    if not page:
        return q3h.Cache(device, n, kvh, hd, positions, fmt, layers=layers)
    cache = paged(device, n, kvh, hd, positions, fmt, page, layers)
    scatter(cache, held, page, rng)
    return cache


# ---------------------------------------------------------------------------
# rows written and read


@pytest.mark.parametrize("fmt,page", [(N, 0), (N, 32), (F, 64), (H, 32), (Q, 128)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rope", list(ROPES))
@pytest.mark.parametrize("tree", [False, True])
def test_append_rounds_the_definition(device, fmt, page, hd, rope, tree):
    """Normed, turned and stored rows: q within half a step of f32, what the
    cache holds equal to the format of the f32 row."""
    print(f"append fmt {fmt} page {page} hd {hd} rope {rope} tree {tree}", flush=True)
    rng = np.random.default_rng(hd + 7 * fmt)
    n, rows, heads, kvh, P = 3, 13, 6, 3, 700
    lens, counts = np.array([0, 640, 31]), np.array([13, 7, 0])
    r = ROPES[rope]
    table, freq, mag, rot, inter = None, None, 1.0, hd, False
    if r is not None:
        rot = r.get("rot", hd)
        rot = int(rot * hd) if isinstance(rot, float) else rot
        inter = r.get("interleaved", False)
        table = q3h.Rope(device, hd, P, 1e4, rot_dim=rot, interleaved=inter,
                         scaling=r.get("scaling"))
        freq, mag = ref.frequencies(rot, 1e4, r.get("scaling"))
    cache = a_cache(device, n, kvh, hd, P, fmt, page, lens + counts, rng, layers=2)
    qkv = rng.standard_normal((n, rows, (heads + 2 * kvh) * hd + 8)).astype(np.float32)
    qkv *= np.exp(rng.standard_normal((n, rows, 1))).astype(np.float32)
    norm = r is not None and rope != "pairs"
    qn = (1 + 0.2 * rng.standard_normal(hd)).astype(np.float32)
    kn = np.exp(rng.standard_normal(hd)).astype(np.float32)
    parents = random_tree(rng, n, rows) if tree else None
    t = dev_f(qkv)
    a, b = heads * hd, (heads + kvh) * hd
    out = torch.full((n, rows, heads, hd), 7.0, device="cuda")
    got = cache.append(t[..., a:b], t[..., b:b + kvh * hd], dev_i(lens), counts=dev_i(counts),
                       parents=None if parents is None else dev_i(parents), q=t[..., :a],
                       q_out=out, rope=table, q_norm=dev_f(qn) if norm else None,
                       k_norm=dev_f(kn) if norm else None, layer=1)
    assert got is out
    k = torch.full((n, rows, kvh, hd), 7.0, device="cuda")
    v = k.clone()
    cache.read(k, v, starts=dev_i(lens), counts=dev_i(counts), layer=1)
    for layer in (0, 1):
        for s in range(n):
            before = torch.full((n, max(1, lens[s]), kvh, hd), 7.0, device="cuda")
            cache.read(before, None, counts=dev_i(lens * (np.arange(n) == s)), layer=layer)
            assert not before[s, :lens[s]].any()
    out, k, v = host(out), host(k), host(v)
    for s in range(n):
        assert (out[s, counts[s]:] == 7).all() and (k[s, counts[s]:] == 7).all()
        for i in range(counts[s]):
            x = qkv[s, i].astype(np.float64)
            q0, k0 = x[:a].reshape(heads, hd), x[a:b].reshape(kvh, hd)
            if norm:
                q0, k0 = ref.normed(q0, qn.astype(np.float64), float(np.float32(1e-6))), \
                    ref.normed(k0, kn.astype(np.float64), float(np.float32(1e-6)))
            if table is not None:
                depth = len(ref.path(None if parents is None else parents[s], i)) - 1
                q0 = ref.turned(q0, lens[s] + depth, rot, inter, freq, mag)
                k0 = ref.turned(k0, lens[s] + depth, rot, inter, freq, mag)
            # one rounding to f32; 64-bit sums add 1e-13 of the head's largest
            tol = U * np.abs(q0) + 1e-13 * np.abs(q0).max()
            assert (np.abs(out[s, i] - q0) <= tol).all()
            np.testing.assert_array_equal(k[s, i], pref.stored(k0.astype(np.float32), fmt))
            v0 = qkv[s, i, b:b + kvh * hd].reshape(kvh, hd)
            np.testing.assert_array_equal(v[s, i], pref.stored(v0, fmt))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [9, 1100])
def test_rows_of_extreme_values(device, hd, rows):
    """Zeros, the smallest and largest values, infinities and NaN, groups of zeros and
    of far smaller values beside others."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((rows, hd)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e-44)
    x[2] *= np.float32(3e-39)
    x[3] = np.float32(3.3e38) * np.sign(x[3])
    x[4, 5] = np.inf
    x[5, 63] = -np.inf
    x[6, 0] = np.nan
    x[7, 32:] *= np.float32(1e-3)
    x[7, :32] = 0
    x[8, :] = 0
    x[8, 9] = np.float32(1e-45)
    # values at the border between two elements: whole numbers of half steps
    x[9:60] = rng.integers(-14, 15, (len(x[9:60]), hd)).astype(np.float32) / 2
    x[9:60, 0] = 7
    cache = q3h.Cache(device, 1, 1, hd, rows + 5, N)
    r = dev_f(x[None, :, None])
    cache.append(r, r, dev_i([0]))
    k, v = torch.zeros_like(r), torch.zeros_like(r)
    cache.read(k, v)
    want = pref.stored(x, N)
    np.testing.assert_array_equal(host(k)[0, :, 0], want)
    np.testing.assert_array_equal(host(v)[0, :, 0], want)


@pytest.mark.parametrize("fmt", [F, H, Q, N])
@pytest.mark.parametrize("hd", [64, 128])
def test_append_of_any_heads_and_distances(device, fmt, hd):
    """Head counts that fill a wave's places or not, rows between 16-byte boundaries,
    many rows of a kind."""
    rng = np.random.default_rng(31)
    for heads, kvh, n, rows in ((0, 1, 1, 3), (5, 5, 2, 2), (9, 3, 1, 7), (33, 11, 1, 2),
                                (2, 1, 3, 500)):
        print(f"heads {heads} kv {kvh} rows {n} x {rows}", flush=True)
        width = (heads + 2 * kvh) * hd + 3
        x = rng.standard_normal((n, rows, width)).astype(np.float32)
        t = dev_f(x)
        cache = paged(device, n, kvh, hd, rows + 40, fmt, 32)
        lens = dev_i([37] * n)
        cache.reserve(dev_i([0] * n), rows + 40, counts=dev_i([37 + rows] * n))
        q = t[..., 1:1 + heads * hd] if heads else None
        a = 1 + heads * hd
        out = cache.append(t[..., a:a + kvh * hd], t[..., a + kvh * hd:a + 2 * kvh * hd], lens, q=q)
        if heads:
            assert torch.equal(out.view(n, rows, -1), q)
        k = torch.zeros((n, rows, kvh, hd), device="cuda")
        v = torch.zeros_like(k)
        cache.read(k, v, starts=lens)
        rows_k = x[..., a:a + kvh * hd].reshape(n, rows, kvh, hd)
        rows_v = x[..., a + kvh * hd:a + 2 * kvh * hd].reshape(n, rows, kvh, hd)
        np.testing.assert_array_equal(host(k), pref.stored(rows_k, fmt))
        np.testing.assert_array_equal(host(v), pref.stored(rows_v, fmt))


AXES = {
    "dealt": [i % 3 if i < 60 else 0 for i in range(64)],
    "parts": [0] * 24 + [1] * 20 + [2] * 20,
    "four": [i % 4 for i in range(64)],
    "one": [0] * 64,
}


@pytest.mark.parametrize("axes", list(AXES))
@pytest.mark.parametrize("rot,interleaved", [(128, False), (64, True), (20, False), (20, True)])
@pytest.mark.parametrize("fmt,page", [(F, 0), (N, 64)])
def test_positions_on_several_axes(device, axes, rot, interleaved, fmt, page):
    rng = np.random.default_rng(41)
    n, rows, heads, kvh, hd, P = 3, 9, 4, 2, 128, 300
    pairs = AXES[axes][:rot // 2]
    k_axes = max(pairs) + 1
    table = q3h.Rope(device, hd, P, 1e4, rot_dim=rot, interleaved=interleaved, axes=pairs)
    freq, mag = ref.frequencies(rot, 1e4)
    lens, counts = np.array([0, 100, 250]), np.array([9, 4, 7])
    places = rng.integers(0, P, (k_axes, n, rows)).astype(np.int32)
    places[0, 0, 1], places[k_axes - 1, 0, 2] = -1, P  # no such positions
    places[k_axes - 1, 1, 0], places[0, 1, 3] = 2 ** 31 - 1, -2 ** 31
    places[0, 0, 0], places[k_axes - 1, 0, 3] = 0, P - 1
    x = rng.standard_normal((n, rows, heads + 2 * kvh, hd)).astype(np.float32)
    t = dev_f(x)
    cache = a_cache(device, n, kvh, hd, P, fmt, page, lens + counts, rng)
    out = torch.full((n, rows, heads, hd), 7.0, device="cuda")
    cache.append(t[:, :, heads:heads + kvh].contiguous(), t[:, :, heads + kvh:].contiguous(),
                 dev_i(lens), counts=dev_i(counts), q=t[:, :, :heads].contiguous(), q_out=out,
                 rope=table, positions=dev_i(places))
    k = torch.zeros((n, rows, kvh, hd), device="cuda")
    v = torch.zeros_like(k)
    cache.read(k, v, starts=dev_i(lens), counts=dev_i(counts))
    out, k, v = host(out), host(k), host(v)
    for s in range(n):
        assert (out[s, counts[s]:] == 7).all()
        for i in range(counts[s]):
            at = places[:, s, i]
            if (at < 0).any() or (at >= P).any():
                assert np.isnan(out[s, i]).all() and not k[s, i].any() and not v[s, i].any()
                continue
            y = pref.turned(x[s, i].astype(np.float64), at, pairs, rot, interleaved, freq, mag)
            tol = U * np.abs(y[:heads]) + 1e-13 * np.abs(y).max()
            assert (np.abs(out[s, i] - y[:heads]) <= tol).all()
            np.testing.assert_array_equal(
                k[s, i], pref.stored(y[heads:heads + kvh].astype(np.float32), fmt))
            np.testing.assert_array_equal(v[s, i], pref.stored(x[s, i, heads + kvh:], fmt))
    # without positions all axes have the row's own
    plain = q3h.Rope(device, hd, P, 1e4, rot_dim=rot, interleaved=interleaved)
    q = t[:, :, :heads].contiguous()
    kv = t[:, :, heads:heads + kvh].contiguous()
    a = cache.append(kv, kv, dev_i(lens), counts=dev_i([9, 9, 9] if not page else counts), q=q,
                     q_out=torch.zeros_like(q), rope=table)
    b = cache.append(kv, kv, dev_i(lens), counts=dev_i([9, 9, 9] if not page else counts), q=q,
                     q_out=torch.zeros_like(q), rope=plain)
    assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# attention


ATTEND = [
    # (fmt, hd, heads, kv_heads, rows, lens, tree)
    (N, 128, 16, 8, 1, [0], False),
    (N, 128, 16, 8, 1, [1, 200, 31], False),
    (N, 64, 4, 2, 1, [63, 64, 65, 500], False),
    (N, 64, 6, 2, 5, [7, 0, 90], True),
    (N, 128, 4, 4, 17, [15, 1000], True),
    (N, 64, 8, 1, 64, [33, 2], True),
    (N, 128, 16, 4, 33, [127, 640], True),
    (N, 128, 28, 4, 11, [1, 95, 350], True),
    (N, 128, 2, 1, 100, [40, 0], False),
    (N, 64, 3, 1, 129, [5, 77], False),
    (N, 128, 8, 2, 70, [300, 1], False),
    (N, 128, 2, 1, 1, [4100, 2000], False),
    (N, 64, 2, 1, 9, [4500], True),
    (N, 128, 8, 2, 300, [900, 350, 0], False),
    (N, 128, 8, 8, 2, [900 - 13 * i for i in range(50)], True),
    (N, 64, 4, 1, 64, [2000, 100, 1500, 30], True),
    (F, 128, 16, 8, 1, [0, 300, 31], False),
    (F, 64, 3, 3, 2, [95, 200], True),
    (F, 128, 4, 2, 64, [1100], True),
    (H, 128, 16, 8, 1, [63, 64, 65], False),
    (H, 64, 8, 2, 300, [900, 350, 0], False),
    (H, 128, 2, 1, 9, [4500], True),
    (Q, 128, 16, 4, 33, [127, 640], True),
    (Q, 128, 2, 1, 1, [4100, 2000], False),
    (Q, 64, 3, 1, 129, [5, 77], False),
]


@pytest.mark.parametrize("case,page", [(i, page) for i, c in enumerate(ATTEND)
                                       for page in (0, 32, 64, 256) if page or c[0] == N])
def test_attend_matches_float64(device, case, page):
    check_attend(device, ATTEND[case], page, 100 + case)


# more sequences than a wave has lanes, and heads of more groups of rows than that
LARGE = [
    (N, 64, 4, 2, 1, [2500 - 7 * i for i in range(70)], False),
    (N, 128, 4, 2, 3, [1200 - 9 * i for i in range(130)], True),
    (N, 64, 2, 1, 2100, [100], False),
    (H, 64, 2, 1, 4200, [30], False),
    (Q, 64, 8, 1, 1200, [300, 0], False),
    (F, 64, 4, 1, 700, [0, 900, 20], False),
]


@pytest.mark.parametrize("page", [0, 32])
@pytest.mark.parametrize("case", range(len(LARGE)))
def test_attend_of_many(device, case, page):
    check_attend(device, LARGE[case], page, 200 + case)


def check_attend(device, case, page, seed):
    fmt, hd, heads, kvh, rows, lens, tree = case
    print("attend", case, page, flush=True)
    rng = np.random.default_rng(seed)
    n, P = len(lens), max(lens) + rows + 3
    lens = np.array(lens)
    counts = np.array([max(1, rows - i * 3) for i in range(n)])
    k = rng.standard_normal((n, P, kvh, hd)).astype(np.float32) * \
        np.exp(0.5 * rng.standard_normal((kvh, hd))).astype(np.float32)
    v = rng.standard_normal((n, P, kvh, hd)).astype(np.float32)
    q = rng.standard_normal((n, rows, heads, hd)).astype(np.float32) * 2
    parents = random_tree(rng, n, rows) if tree else None
    cache = a_cache(device, n, kvh, hd, P, fmt, page, lens + counts, rng)
    fill(cache, k, v, lens + counts)
    wide = np.zeros((n, rows, heads * hd + 12), np.float32)  # rows further apart
    wide[..., :heads * hd] = q.reshape(n, rows, -1)
    out = torch.full((n, rows, heads, hd), 7.0, device="cuda")
    args = dict(counts=dev_i(counts), parents=None if parents is None else dev_i(parents))
    cache.attend(dev_f(wide)[..., :heads * hd], dev_i(lens), int(lens.max()), out=out, **args)
    held = pref.stored(k, fmt).astype(np.float64), pref.stored(v, fmt).astype(np.float64)
    want, bound = ref.attention(q.astype(np.float64), *held, lens, counts, parents, hd ** -0.5)
    got = host(out)
    for s in range(n):
        assert (got[s, counts[s]:] == 7).all()
        d = np.abs(got[s, :counts[s]] - want[s, :counts[s]])
        worst = float((d / np.maximum(bound[s, :counts[s]], 1e-300)).max())
        print(f"sequence {s}: {d.max():.2e}, {worst:.2e} of the bound", flush=True)
        assert worst <= 1
    if page:
        # the same as over a cache in one piece, bit for bit
        whole = q3h.Cache(device, n, kvh, hd, P, fmt)
        fill(whole, k, v, lens + counts)
        same = torch.full((n, rows, heads, hd), 7.0, device="cuda")
        whole.attend(dev_f(wide)[..., :heads * hd], dev_i(lens), int(lens.max()), out=same, **args)
        assert torch.equal(out, same)


@pytest.mark.parametrize("fmt,page", [(N, 0), (N, 32), (F, 32), (H, 32), (Q, 32)])
@pytest.mark.parametrize("heads", [2, 32])
def test_unseen_rows_do_not_reach_a_row(device, fmt, page, heads):
    """Infinities and NaN in siblings' positions, behind the rows, in the rest of the last
    page and in pages of others."""
    rng = np.random.default_rng(21)
    hd, rows, P, length = 128, 12, 90, 37
    k = rng.standard_normal((1, P, 2, hd)).astype(np.float32)
    v = rng.standard_normal((1, P, 2, hd)).astype(np.float32)
    parents = np.array([[-1, 0, 0, 1, 2, 3, 4, -1, 7, 8, 9, 10]], np.int32)
    for r in (2, 4, 6):  # a branch of its own: 0 -> 2 -> 4 -> 6
        k[0, length + r, :, r] = np.nan
        v[0, length + r, :, 3 * r] = np.inf
    k[0, length + rows:] = np.nan
    v[0, length + rows:, :, ::3] = -np.inf
    q = rng.standard_normal((1, rows, heads, hd)).astype(np.float32)
    cache = a_cache(device, 2 if page else 1, 2, hd, P, fmt, page, [P, P] if page else [P], rng)
    if page:  # (the other sequence: NaN throughout)
        nan = np.full((2, P, 2, hd), np.nan, np.float32)
        fill(cache, nan, nan, [P, P])
    fill(cache, k, v, [P])
    out = host(cache.attend(dev_f(q), dev_i([length]), length, parents=dev_i(parents)))
    clean = [0, 1, 3, 5, 7, 8, 9, 10, 11]
    assert np.isnan(out[0, [2, 4, 6]]).all()
    kk, vv = [np.nan_to_num(pref.stored(x, fmt), nan=0, posinf=0, neginf=0).astype(np.float64)
              for x in (k, v)]
    want, bound = ref.attention(q.astype(np.float64), kk, vv, [length], [rows], parents, hd ** -0.5)
    assert (np.abs(out - want)[0, clean] <= bound[0, clean]).all()
    # a chain sees all that came before it
    out = host(cache.attend(dev_f(q), dev_i([length]), length))
    assert np.isfinite(out[0, :2]).all() and np.isnan(out[0, 2:]).all()


@pytest.mark.parametrize("size", [2.0 ** -110, 2.0 ** -70, 2.0 ** -50, 2.0 ** 45, 2.0 ** 70, 2.0 ** 110])
@pytest.mark.parametrize("heads", [1, 20])
@pytest.mark.parametrize("hd", [64, 128])
def test_attend_values_of_any_size(device, size, heads, hd):
    rng = np.random.default_rng(26)
    rows, P, length = 3, 300, 290
    k = rng.standard_normal((1, P, 1, hd)).astype(np.float32)
    v = (rng.standard_normal((1, P, 1, hd)) * size).astype(np.float32)
    v[0, 64:96] = 0
    v[0, 200:240] *= 2.0 ** -16
    q = rng.standard_normal((1, rows, heads, hd)).astype(np.float32)
    cache = q3h.Cache(device, 1, 1, hd, P, N)
    fill(cache, k, v, [length + rows])
    held = pref.stored(k, N).astype(np.float64), pref.stored(v, N).astype(np.float64)
    want, bound = ref.attention(q.astype(np.float64), *held, [length], [rows], None, hd ** -0.5)
    out = host(cache.attend(dev_f(q), dev_i([length]), length))
    ratio = np.abs(out - want) / bound
    print(ratio.max(), flush=True)
    assert (ratio <= 1).all()


@pytest.mark.parametrize("heads", [2, 24])
def test_outlying_channels_cost_no_precision(device, heads):
    """Keys and values with a few elements hundreds of times the others: the products stay
    those of f32 over what the cache holds, relative to a row's largest element."""
    rng = np.random.default_rng(27)
    hd, rows, P, length = 128, 20, 400, 380
    k = rng.standard_normal((1, P, 1, hd)).astype(np.float32)
    v = rng.standard_normal((1, P, 1, hd)).astype(np.float32)
    k[..., 17] *= 200
    v[..., 99] *= 500
    q = rng.standard_normal((1, rows, heads, hd)).astype(np.float32)
    q[..., 17] /= 200
    cache = q3h.Cache(device, 1, 1, hd, P, N)
    fill(cache, k, v, [length + rows])
    held = pref.stored(k, N).astype(np.float64), pref.stored(v, N).astype(np.float64)
    want, bound = ref.attention(q.astype(np.float64), *held, [length], [rows], None, hd ** -0.5)
    out = host(cache.attend(dev_f(q), dev_i([length]), length))
    ratio = np.abs(out - want) / bound
    print(ratio.max(), flush=True)
    assert (ratio <= 1).all()


@pytest.mark.parametrize("fmt,page", [(N, 0), (N, 32), (H, 32), (F, 64), (Q, 32)])
@pytest.mark.parametrize("hd", [64, 128])
def test_keep_moves_the_path_forward(device, fmt, page, hd):
    rng = np.random.default_rng(8)
    n, rows, kvh, layers, P = 4, 40, 3, 3, 200
    lens = np.array([20, 31, 100, 0])
    cache = a_cache(device, n, kvh, hd, P, fmt, page, lens + rows, rng, layers=layers)
    x = [rng.standard_normal((n, 160, kvh, hd)).astype(np.float32) for _ in range(2 * layers)]
    for layer in range(layers):
        fill(cache, x[2 * layer], x[2 * layer + 1], lens + rows, layer=layer)
    kept = np.zeros((n, rows), np.int32)
    lists = [[0, 3, 4, 11, 12, 13, 35], list(range(1, 40)), [39], [2, 1]]  # the last: not a path
    for b, one in enumerate(lists):
        kept[b, :len(one)] = one
    cache.keep(dev_i(lens), dev_i(kept), dev_i([len(one) for one in lists]))
    for layer in range(layers):
        k = torch.zeros((n, 160, kvh, hd), device="cuda")
        v = torch.zeros_like(k)
        cache.read(k, v, counts=dev_i(lens + rows), layer=layer)
        for got, rows_in in ((host(k), x[2 * layer]), (host(v), x[2 * layer + 1])):
            want = pref.stored(rows_in, fmt)
            for b, one in enumerate(lists):
                now = want[b].copy()
                if b != 3:
                    now[lens[b]:lens[b] + len(one)] = want[b, lens[b] + np.array(one)]
                np.testing.assert_array_equal(got[b, :lens[b] + rows], now[:lens[b] + rows])


# ---------------------------------------------------------------------------
# pages


def state_of(cache):
    return [t.cpu().numpy() for t in cache.page_state()]


def check_state(cache, model):
    table, counts, refs = state_of(cache)
    np.testing.assert_array_equal(counts, [len(held) for held in model.lists])
    np.testing.assert_array_equal(table, model.table())
    np.testing.assert_array_equal(refs, model.refs())


@pytest.mark.parametrize("seed", range(6))
def test_tables_follow_the_definition(device, seed):
    """Reserve, fork, release and compact in any order, with few pages (they run out),
    arguments out of range among them, against lists, the contents against a copy of
    every sequence."""
    rng = np.random.default_rng(seed)
    n = int(rng.choice([1, 3, 9, 40, 70]))
    page = int(rng.choice([32, 64]))
    P = int(rng.integers(1, 500))
    pages = int(rng.integers(max(2, n // 2), n * (-(-P // page)) + 2))
    print(f"seed {seed}: {n} sequences of {P}, {pages} pages of {page}", flush=True)
    kvh, hd, layers, fmt = 2, 64, 2, [F, H, Q, N][seed % 4]
    cache = q3h.Cache(device, n, kvh, hd, P, fmt, layers=layers, pages=pages, page_positions=page)
    model = pref.Pages(n, pages, page, P)
    # what is known of the contents: [sequence] -> rows [position][layer][part]
    known = [np.full((P, layers, 2), np.nan) for _ in range(n)]
    stamp = 0
    for turn in range(40):
        what = rng.choice(["reserve", "reserve", "reserve", "fork", "release", "compact"])
        m = int(rng.integers(1, n + 1))
        room = [len(held) * page for held in model.lists]
        if what == "reserve":
            rows = int(rng.integers(1, P + 1)) if rng.random() < 0.5 else 1
            lens = np.array([rng.integers(0, min(P, r) + 1) for r in room[:m]])
            counts = rng.integers(0, rows + 1, m)
            odd = rng.random(m) < 0.1
            lens[odd] = rng.choice([-1, P, P + 1, 2 ** 31 - 1], odd.sum())
            ok = torch.full((m,), 9, dtype=torch.int32, device="cuda")
            cache.reserve(dev_i(lens), rows, counts=dev_i(counts), ok=ok)
            want, copies = model.reserve(lens.tolist(), counts.tolist())
            np.testing.assert_array_equal(ok.cpu().numpy(), want)
            # rows into what was reserved: a value of their own, exact in every format
            good = np.array(want) * counts
            good[~((lens >= 0) & (lens <= P))] = 0
            if good.any():
                stamp += 1
                for layer in range(layers):
                    k = np.zeros((m, rows, kvh, hd), np.float32)
                    k[:] = (1785 * (2 * stamp + layer))
                    cache.append(dev_f(k), dev_f(-k), dev_i(lens), counts=dev_i(good), layer=layer)
                for b in range(m):
                    if good[b]:
                        known[b][lens[b]:lens[b] + good[b]] = [
                            [1785 * (2 * stamp + layer) * s for s in (1, -1)] for layer in range(layers)]
                        known[b][lens[b] + good[b]:] = np.nan
        elif what == "fork":
            sources = rng.integers(-1, n, m)
            lens = np.array([rng.integers(0, min(P, room[s]) + 1) if s >= 0 else 5 for s in sources])
            odd = rng.random(m) < 0.1
            sources[odd] = rng.choice([-2, n, 2 ** 31 - 1], odd.sum())
            lens[rng.random(m) < 0.05] = -3
            was = [x.copy() for x in known]
            cache.fork(dev_i(sources), dev_i(lens))
            before = [list(x) for x in model.lists]
            model.fork(sources.tolist(), lens.tolist())
            for b in range(m):
                s = sources[b]
                if s == -1:
                    known[b][:] = np.nan
                elif 0 <= s < n and 0 <= lens[b] <= len(before[s]) * page:
                    known[b][:] = np.nan
                    known[b][:lens[b]] = was[s][:lens[b]]
        elif what == "release":
            lens = rng.integers(-1, P + 40, m)
            cache.release(dev_i(lens))
            model.release(lens.tolist())
            for b in range(m):
                known[b][len(model.lists[b]) * page:] = np.nan
        else:
            used = cache.compact()
            assert used.item() == model.compact()[0]
        check_state(cache, model)
        for layer in range(layers):
            k = torch.zeros((n, P, kvh, hd), device="cuda")
            v = torch.zeros_like(k)
            held = np.array([min(P, len(x) * page) for x in model.lists])
            cache.read(k, v, counts=dev_i(held), layer=layer)
            for part, got in enumerate((host(k), host(v))):
                for b in range(n):
                    want = known[b][:held[b], layer, part]
                    sure = np.isfinite(want)
                    exact = pref.stored(np.repeat(want[sure, None].astype(np.float32), hd, 1), fmt)
                    np.testing.assert_array_equal(got[b, :held[b]][sure],
                                                  np.repeat(exact[:, None], kvh, 1))


@pytest.mark.parametrize("pages,page,n", [(5000, 32, 300), (70000, 32, 5), (9000, 64, 1200)])
def test_large_tables(device, pages, page, n):
    """More pages than a workgroup looks at in one go, more sequences than it has groups."""
    rng = np.random.default_rng(pages)
    P = 4000
    cache = q3h.Cache(device, n, 1, 64, P, N, pages=pages, page_positions=page)
    model = pref.Pages(n, pages, page, P)
    for turn in range(4):
        lens = np.array([rng.integers(0, len(held) * page + 1) for held in model.lists])
        lens = np.minimum(lens, P - 1)
        counts = rng.integers(0, P - lens + 1) // rng.choice([1, 3, 20], n)
        ok = torch.zeros(n, dtype=torch.int32, device="cuda")
        cache.reserve(dev_i(lens), P, counts=dev_i(counts), ok=ok)
        want, _ = model.reserve(lens.tolist(), counts.tolist())
        np.testing.assert_array_equal(ok.cpu().numpy(), want)
        check_state(cache, model)
        lens = rng.integers(0, P, n)
        cache.release(dev_i(lens))
        model.release(lens.tolist())
        sources = rng.integers(-1, n, n)
        lens = np.array([rng.integers(0, len(model.lists[s]) * page + 1) if s >= 0 else 0
                         for s in sources])
        cache.fork(dev_i(sources), dev_i(lens))
        model.fork(sources.tolist(), lens.tolist())
        check_state(cache, model)
        assert cache.compact().item() == model.compact()[0]
        check_state(cache, model)


def test_a_page_that_all_write_to_is_kept_by_the_first(device):
    cache = q3h.Cache(device, 4, 1, 64, 100, H, pages=8, page_positions=32)
    cache.reserve(dev_i([0, 0, 0, 0]), 40, counts=dev_i([40, 0, 0, 0]))
    k = np.arange(40, dtype=np.float32)[None, :, None, None] * np.ones((1, 1, 1, 64), np.float32)
    fill(cache, k, k, [40])
    cache.fork(dev_i([0, 0, 0, 0]), dev_i([40, 40, 40, 32]))
    # one of three: it leaves
    ok = torch.zeros(4, dtype=torch.int32, device="cuda")
    cache.reserve(dev_i([40, 40, 40, 32]), 1, counts=dev_i([0, 1, 0, 0]), ok=ok)
    assert ok.tolist() == [1, 1, 1, 1]
    assert state_of(cache)[0].tolist() == [[0, 1, -1, -1], [0, 2, -1, -1], [0, 1, -1, -1],
                                           [0, -1, -1, -1]]
    # both that are left: the first keeps it, the other gets a copy
    cache.reserve(dev_i([40, 40, 40, 32]), 1, counts=dev_i([1, 0, 1, 0]), ok=ok)
    table, counts, refs = state_of(cache)
    assert table.tolist() == [[0, 1, -1, -1], [0, 2, -1, -1], [0, 3, -1, -1], [0, -1, -1, -1]]
    assert refs.tolist() == [4, 1, 1, 1, 0, 0, 0, 0]
    out = torch.zeros((4, 40, 1, 64), device="cuda")
    cache.read(out, None, counts=dev_i([40, 40, 40, 32]))
    for b in range(4):
        m = 40 if b < 3 else 32
        np.testing.assert_array_equal(host(out)[b, :m], k[0, :m])


def test_shared_pages_are_not_written(device):
    """Rows that would go to a page of two sequences: NaN queries, nothing written;
    a keep whose path would, neither."""
    rng = np.random.default_rng(3)
    cache = q3h.Cache(device, 2, 2, 64, 128, N, pages=8, page_positions=32)
    k = rng.standard_normal((2, 50, 2, 64)).astype(np.float32)
    cache.reserve(dev_i([0, 0]), 50, counts=dev_i([50, 0]))
    fill(cache, k[:1], k[:1], [50])
    cache.fork(dev_i([0, 0]), dev_i([50, 50]))
    q = dev_f(rng.standard_normal((2, 20, 2, 64)))
    new = dev_f(rng.standard_normal((2, 20, 2, 64)))
    out = host(cache.append(new, new, dev_i([40, 50]), counts=dev_i([10, 14]), q=q,
                            q_out=torch.zeros_like(q)))
    assert np.isnan(out[0, :10]).all() and not out[0, 10:].any()
    assert np.isnan(out[1, :14]).all() and not out[1, 14:].any()
    kept = np.tile(np.arange(20) + 1, (2, 1))
    cache.keep(dev_i([40, 40]), dev_i(kept), dev_i([3, 3]))
    got = torch.zeros((2, 50, 2, 64), device="cuda")
    cache.read(got, None)
    for b in range(2):
        np.testing.assert_array_equal(host(got)[b], pref.stored(k[0], N))
    # its own page: written
    ok = torch.zeros(2, dtype=torch.int32, device="cuda")
    cache.reserve(dev_i([50, 50]), 20, counts=dev_i([0, 20]), ok=ok)
    assert ok.tolist() == [1, 1]
    assert np.isfinite(host(cache.append(new, new, dev_i([0, 50]), counts=dev_i([0, 20]), q=q,
                                         q_out=torch.zeros_like(q)))).all()
    cache.read(got, None)
    np.testing.assert_array_equal(host(got)[0], pref.stored(k[0], N))


@pytest.mark.parametrize("fmt", [F, H, Q, N])
def test_sequences_without_pages(device, fmt):
    """Positions behind a sequence's pages: NaN where they are asked for, nothing
    written; the sequences beside it as ever."""
    rng = np.random.default_rng(9)
    cache = q3h.Cache(device, 4, 2, 64, 200, fmt, pages=6, page_positions=32)
    k = rng.standard_normal((4, 40, 2, 64)).astype(np.float32)
    cache.reserve(dev_i([0] * 4), 40, counts=dev_i([40, 0, 31, 0]))
    fill(cache, k, k, [40, 0, 31, 0])
    q = dev_f(rng.standard_normal((4, 3, 2, 64)))
    lens = dev_i([37, 0, 30, 200])
    new = dev_f(rng.standard_normal((4, 3, 2, 64)))
    out = host(cache.append(new, new, lens, q=q))
    assert np.isfinite(out[0]).all() and np.isnan(out[1:]).all()
    got = torch.zeros((4, 3, 2, 64), device="cuda")
    cache.read(got, None, starts=lens)
    assert np.isfinite(host(got)[0]).all() and np.isnan(host(got)[1:]).all()
    o = host(cache.attend(q, lens, 200))
    assert np.isfinite(o[0]).all() and np.isnan(o[1:]).all()
    whole = torch.zeros((4, 31, 2, 64), device="cuda")
    cache.read(whole, None, counts=dev_i([31, 0, 31, 0]))
    np.testing.assert_array_equal(host(whole)[2], pref.stored(k[2, :31], fmt))


@pytest.mark.parametrize("fmt", [F, H, Q, N])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("pages", [(0, 32), (64, 0), (32, 256), (256, 32), (0, 0)])
def test_copies_between_caches(device, fmt, hd, pages):
    rng = np.random.default_rng(17)
    n, m, kvh, layers, P = 5, 6, 3, 2, 300
    held = np.array([300, 0, 33, 100, 1, 257])
    src = a_cache(device, m, kvh, hd, P, fmt, pages[0], held, rng, layers=layers)
    sources = np.array([5, -1, 0, 2, 7])
    lens = np.array([257, 10, 290, 20, 5])
    if pages[0]:
        sources[3], lens[3] = 4, 40  # behind its page of 32; of the larger ones zeros too
    dst = a_cache(device, n, kvh, hd, P + 20, fmt, pages[1], [260, 30, 320, 64, 9], rng,
                  layers=layers)
    x = [rng.standard_normal((m, P, kvh, hd)).astype(np.float32) for _ in range(2 * layers)]
    y = rng.standard_normal((n, 320, kvh, hd)).astype(np.float32)
    room = np.array([260, 30, 320, 64, 9])
    for layer in range(layers):
        fill(src, x[2 * layer], x[2 * layer + 1], held, layer=layer)
        fill(dst, y, y, room, layer=layer)
    dst.copy(src, dev_i(sources), dev_i(lens))
    for layer in range(layers):
        k = torch.zeros((n, 320, kvh, hd), device="cuda")
        v = torch.zeros_like(k)
        dst.read(k, v, counts=dev_i(room), layer=layer)
        for got, rows in ((host(k), x[2 * layer]), (host(v), x[2 * layer + 1])):
            for b in range(n):
                want = pref.stored(y[b, :room[b]], fmt)
                copied = b in (0, 2) or (b == 3 and pages[0] != 32)
                if copied:
                    want[:lens[b]] = pref.stored(rows[sources[b], :lens[b]], fmt)
                    want[held[sources[b]]:lens[b]] = 0
                np.testing.assert_array_equal(got[b, :room[b]], want)


def test_copies_of_many_sequences_leave_shared_pages(device):
    rng = np.random.default_rng(19)
    n, P = 150, 90
    src = q3h.Cache(device, n, 1, 64, P, N)
    dst = q3h.Cache(device, n, 1, 64, P, N, pages=3 * n, page_positions=32)
    x = rng.standard_normal((n, P, 1, 64)).astype(np.float32)
    fill(src, x, -x, [P] * n)
    dst.reserve(dev_i([0] * n), P)
    y = np.full((n, P, 1, 64), 3, np.float32)
    fill(dst, y, y, [P] * n)
    # sequence 1 shares the first page of sequence 0
    sources = np.arange(n)
    sources[1] = 0
    lens = np.full(n, P)
    lens[1] = 32
    dst.fork(dev_i(sources), dev_i(lens))
    lens = rng.integers(0, P + 1, n)
    lens[:2] = [P, 32]
    order = rng.permutation(n)
    dst.copy(src, dev_i(order), dev_i(lens))
    got = torch.zeros((n, P, 1, 64), device="cuda")
    dst.read(got, None, counts=dev_i([P, 32] + [P] * (n - 2)))
    for b in range(n):
        want = pref.stored(y[b], N)
        want[:lens[b]] = pref.stored(x[order[b], :lens[b]], N)
        if b < 2:
            want[:32] = pref.stored(y[b, :32], N)
        m = 32 if b == 1 else P
        np.testing.assert_array_equal(host(got)[b, :m], want[:m])


# ---------------------------------------------------------------------------
# together


@pytest.mark.parametrize("fmt", [H, N])
def test_a_server_of_beams(device, fmt):
    """Prompts with positions on three axes, forked into beams that write tokens of
    their own, are reordered and dropped while the pages are moved together; drafted
    trees and kept paths on what is left: every attention against float64 over the rows
    that its sequence has seen."""
    rng = np.random.default_rng(51)
    hd, heads, kvh, P, page, beams = 64, 4, 2, 260, 32, 4
    n, prompts = 8, 2
    cache = q3h.Cache(device, n, kvh, hd, P, fmt, pages=30, page_positions=page)
    pairs = [i % 3 if i < 30 else 0 for i in range(32)]
    rope = q3h.Rope(device, hd, P, 1e4, axes=pairs)
    freq, mag = ref.frequencies(hd, 1e4)
    seen = [([], []) for _ in range(n)]  # stored keys and values of each sequence
    lens = np.zeros(n, int)

    def rows_in(counts, rows, parents=None):
        """Rows of all sequences: reserved, appended, attended; returns the outputs."""
        ok = torch.zeros(n, dtype=torch.int32, device="cuda")
        cache.reserve(dev_i(lens), rows, counts=dev_i(counts), ok=ok)
        assert ok.tolist() == [1] * n
        x = rng.standard_normal((n, rows, heads + 2 * kvh, hd)).astype(np.float32)
        places = rng.integers(0, P, (3, n, rows))
        t = dev_f(x)
        q = cache.append(t[:, :, heads:heads + kvh].contiguous(),
                         t[:, :, heads + kvh:].contiguous(), dev_i(lens), counts=dev_i(counts),
                         q=t[:, :, :heads].contiguous(), rope=rope, positions=dev_i(places),
                         parents=None if parents is None else dev_i(parents))
        out = host(cache.attend(q, dev_i(lens), P, counts=dev_i(counts),
                                parents=None if parents is None else dev_i(parents)))
        for b in range(n):
            ks, vs = [list(z) for z in seen[b]]
            qs = []
            for i in range(counts[b]):
                y = pref.turned(x[b, i].astype(np.float64), places[:, b, i], pairs, hd, False,
                                freq, mag)
                qs.append(y[:heads].astype(np.float32).astype(np.float64))
                ks.append(pref.stored(y[heads:heads + kvh].astype(np.float32), fmt))
                vs.append(pref.stored(x[b, i, heads + kvh:], fmt))
            seen[b] = (ks, vs)
            if not counts[b]:
                continue
            want, bound = ref.attention(
                np.array(qs)[None], np.array(ks, np.float64)[None], np.array(vs, np.float64)[None],
                [lens[b]], [counts[b]], None if parents is None else parents[b:b + 1], hd ** -0.5)
            d = np.abs(out[b, :counts[b]] - want[0])
            assert (d <= bound[0] + 4 * U * np.abs(want[0])).all(), (b, (d / bound[0]).max())

    counts = np.array([50, 75] + [0] * (n - 2))
    rows_in(counts, 75)
    lens += counts
    # four beams of each prompt
    sources = np.arange(n) % prompts
    cache.fork(dev_i(sources), dev_i(lens[sources]))
    seen = [tuple(list(z) for z in seen[s]) for s in sources]
    lens = lens[sources]
    for step in range(3):
        rows_in(np.ones(n, int), 1)
        lens += 1
        sources = rng.integers(0, n, n)  # the beams that go on, any number of times
        if step == 1:
            cut = lens - 3  # and some steps back
            cache.fork(dev_i(sources), dev_i(cut[sources]))
            lens = cut[sources]
        else:
            cache.fork(dev_i(sources), dev_i(lens[sources]))
            lens = lens[sources]
        seen = [tuple(list(z)[:m] for z in seen[s]) for s, m in zip(sources, lens)]
        cache.compact()
    # half of them leave, the others draft trees and keep a path
    gone = np.arange(n) % 2 == 1
    lens[gone] = 0
    seen = [([], []) if gone[b] else seen[b] for b in range(n)]
    cache.release(dev_i(lens))
    cache.compact()
    parents = random_tree(rng, n, 9)
    counts = np.where(gone, 0, 9)
    rows_in(counts, 9, parents)
    kept, kept_counts = np.zeros((n, 9), int), np.zeros(n, int)
    for b in range(n):
        if not gone[b]:
            path = ref.path(parents[b], 8)[::-1]
            kept[b, :len(path)], kept_counts[b] = path, len(path)
            seen[b] = tuple(z[:lens[b]] + [z[lens[b] + r] for r in path] for z in seen[b])
    cache.keep(dev_i(lens), dev_i(kept), dev_i(kept_counts))
    lens += kept_counts
    rows_in(np.where(gone, 0, 2), 2)
    table, held, refs = state_of(cache)
    assert (refs.sum() == held.sum()) and (np.sort(table[table >= 0])[-1] < 30)


def test_captured_calls_follow_lengths_and_pages_on_the_device(device):
    """A captured step (fork, reserve, append, attend, compact) replayed over lengths, sources
    and rows that change between the replays, with eager calls in between, against the
    same step made eagerly on a cache of the same history."""
    rng = np.random.default_rng(61)
    n, rows, heads, kvh, hd, P = 6, 3, 4, 2, 128, 400
    made = [q3h.Cache(device, n, kvh, hd, P, N, pages=50, page_positions=32) for _ in range(2)]
    first = rng.standard_normal((n, 200, kvh, hd)).astype(np.float32)
    start = np.array([200, 10, 64, 0, 31, 150])
    for c in made:
        c.reserve(dev_i([0] * n), 200, counts=dev_i(start))
        fill(c, first, first, start)
    sources, keep_to, lens, counts = [torch.zeros(n, dtype=torch.int32, device="cuda")
                                      for _ in range(4)]
    x = torch.zeros((n, rows, heads + 2 * kvh, hd), device="cuda")
    space = torch.zeros(max(1, made[0].attend_workspace(n, rows, heads, P)), dtype=torch.uint8,
                        device="cuda")

    def step(cache, out, ok):
        cache.fork(sources, keep_to)
        cache.reserve(lens, rows, counts=counts, ok=ok)
        q = cache.append(x[:, :, heads:heads + kvh].flatten(2), x[:, :, heads + kvh:].flatten(2),
                         lens, counts=counts, q=x[:, :, :heads].flatten(2))
        cache.attend(q, lens, P, out=out, counts=counts, workspace=space)
        cache.compact(used)

    used = torch.zeros(1, dtype=torch.int32, device="cuda")
    outs = [torch.zeros((n, rows, heads, hd), device="cuda") for _ in range(2)]
    oks = [torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2)]

    def set_inputs(length):
        order = rng.integers(0, n, n)
        cut = np.maximum(0, length[order] - rng.integers(0, 40, n))
        c = rng.integers(0, rows + 1, n)
        sources.copy_(dev_i(order))
        keep_to.copy_(dev_i(cut))
        lens.copy_(dev_i(cut))
        counts.copy_(dev_i(c))
        x.copy_(dev_f(rng.standard_normal(x.shape)))
        return cut + c

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    sources.copy_(torch.arange(n, dtype=torch.int32, device="cuda"))
    keep_to.copy_(dev_i(start))
    lens.copy_(dev_i(start))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step(made[0], outs[0], oks[0])  # (nothing changes: no rows)
        with torch.cuda.graph(graph, stream=side):
            step(made[0], outs[0], oks[0])
    torch.cuda.synchronize()
    length = start
    for turn in range(6):
        length = set_inputs(length)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(made[1], outs[1], oks[1])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(*oks)
        assert oks[0].tolist() == [1] * n
        for a, b in zip(state_of(made[0]), state_of(made[1])):
            np.testing.assert_array_equal(a, b)


def test_calls_on_another_stream(device):
    rng = np.random.default_rng(71)
    cache = q3h.Cache(device, 2, 2, 64, 100, N, pages=9, page_positions=32)
    k = rng.standard_normal((2, 60, 2, 64)).astype(np.float32)
    side = torch.cuda.Stream()
    zero, x, sources, lens = dev_i([0, 0]), dev_f(k), dev_i([1, 1]), dev_i([60, 50])
    out = torch.zeros((2, 60, 2, 64), device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        cache.reserve(zero, 60)
        cache.append(x, x, zero)
        cache.fork(sources, lens)
        cache.read(out, None, counts=lens)
        table, held, refs = cache.page_state()
    side.synchronize()
    want = pref.stored(k, N)
    np.testing.assert_array_equal(host(out)[0], want[1])
    np.testing.assert_array_equal(host(out)[1, :50], want[1, :50])
    assert held.tolist() == [2, 2] and refs.sum().item() == 4


def test_offsets_past_32_bits(device):
    """Pages and rows of a 4-bit cache beyond 4 GiB of one allocation."""
    rng = np.random.default_rng(81)
    kvh, hd, page = 8, 128, 256
    pages = (9 << 30) // (2 * kvh * page * 72 * 4)  # of four layers, 9 GiB
    cache = q3h.Cache(device, 2, kvh, hd, page * (pages // 2), N, layers=4, pages=pages,
                      page_positions=page)
    P = page * (pages // 2)
    cache.reserve(dev_i([0, 0]), P)
    lens = dev_i([P - 70, P - 300])
    rows = rng.standard_normal((2, 60, kvh, hd)).astype(np.float32)
    x = dev_f(rows)
    cache.append(x, -x, lens, layer=3)
    k, v = torch.zeros_like(x), torch.zeros_like(x)
    cache.read(k, v, starts=lens, layer=3)
    np.testing.assert_array_equal(host(k), pref.stored(rows, N))
    np.testing.assert_array_equal(host(v), pref.stored(-rows, N))
    cache.release(dev_i([0, P]))
    assert cache.compact().item() == pages // 2
    got = torch.zeros((2, 60, kvh, hd), device="cuda")
    cache.read(got, None, starts=dev_i([0, P - 300]), counts=dev_i([0, 60]), layer=3)
    np.testing.assert_array_equal(host(got)[1], pref.stored(rows[1], N))
    del cache
    whole = q3h.Cache(device, 1, kvh, hd, 1 << 21, N, layers=2)
    lens = dev_i([(1 << 21) - 80])
    whole.append(x[:1], -x[:1], lens, layer=1)
    whole.read(k[:1], v[:1], starts=lens, layer=1)
    np.testing.assert_array_equal(host(k)[:1], pref.stored(rows[:1], N))
    np.testing.assert_array_equal(host(v)[:1], pref.stored(-rows[:1], N))


def test_empty_calls(device):
    cache = q3h.Cache(device, 2, 2, 64, 100, N, pages=4, page_positions=32)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    cache.reserve(none, 5)
    cache.reserve(dev_i([0, 0]), 0)
    cache.fork(none, none)
    cache.release(none)
    assert cache.compact().item() == 0
    other = q3h.Cache(device, 2, 2, 64, 100, N)
    cache.copy(other, none, none)
    other.copy(cache, dev_i([0, 1]), dev_i([0, 0]))
    x = torch.zeros((2, 0, 2, 64), device="cuda")
    cache.append(x, x, dev_i([0, 0]))
    table, counts, refs = state_of(cache)
    assert (table == -1).all() and not counts.any() and not refs.any()


def test_refusals_of_tensors(device):
    cache = q3h.Cache(device, 2, 2, 64, 100, N, pages=4, page_positions=32)
    whole = q3h.Cache(device, 2, 2, 64, 100, N)
    rope = q3h.Rope(device, 64, 100, 1e4, axes=[i % 3 for i in range(32)])
    x = torch.zeros((2, 3, 2, 64), device="cuda")
    good, wide, host_ints = dev_i([0, 0]), dev_i([[0, 0]]), torch.zeros(2, dtype=torch.int32)
    calls = [
        lambda: whole.reserve(good, 3), lambda: whole.fork(good, good),
        lambda: whole.release(good), lambda: whole.compact(), lambda: whole.page_state(),
        lambda: cache.reserve(dev_i([0, 0, 0]), 3), lambda: cache.reserve(good.long(), 3),
        lambda: cache.reserve(host_ints, 3), lambda: cache.reserve(good, 3, counts=dev_i([0])),
        lambda: cache.reserve(good, 3, ok=dev_f([0, 0])), lambda: cache.fork(good, dev_i([0])),
        lambda: cache.release(wide[:, ::2]), lambda: cache.compact(used=good),
        lambda: cache.copy(cache, good, good), lambda: cache.copy(whole, good, dev_i([0])),
        lambda: cache.copy(q3h.Cache(device, 2, 2, 64, 100, Q), good, good),
        lambda: cache.copy(q3h.Cache(device, 2, 2, 128, 100, N), good, good),
        lambda: cache.append(x, x, good, rope=rope, positions=dev_i(np.zeros((2, 2, 3)))),
        lambda: cache.append(x, x, good, rope=rope, positions=torch.zeros((3, 2, 3), device="cuda")),
        lambda: cache.append(x, x, good, positions=dev_i(np.zeros((1, 2, 3)))),
        lambda: q3h.Rope(device, 64, 100, 1e4, axes=[0] * 31),
        lambda: q3h.Rope(device, 64, 100, 1e4, axes=[4] * 32),
        lambda: q3h.Rope(device, 64, 100, 1e4, axes=[-1] * 32),
        lambda: q3h.Cache(device, 2, 2, 64, 100, N, pages=4, page_positions=16),
        lambda: q3h.Cache(device, 2, 2, 64, 100, 3),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(q3h.Q3HError) as e:
            call()
        assert e.value.code == q3h.E_ARG, i
    with pytest.raises(q3h.Q3HError) as e:
        cache.reserve(good, 101)
    assert e.value.code == q3h.E_CAPACITY
    assert not state_of(cache)[1].any()


def test_destroyed_handles_are_refused(device):
    cache = q3h.Cache(device, 2, 2, 64, 100, N, pages=4, page_positions=32)
    other = q3h.Cache(device, 2, 2, 64, 100, N)
    good = dev_i([0, 0])
    other.destroy()
    with pytest.raises(q3h.Q3HError):
        cache.copy(other, good, good)
    cache.destroy()
    for call in (lambda: cache.reserve(good, 3), lambda: cache.fork(good, good),
                 lambda: cache.release(good), lambda: cache.compact(), lambda: cache.page_state()):
        with pytest.raises(q3h.Q3HError):
            call()
