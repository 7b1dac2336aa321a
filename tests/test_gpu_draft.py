"""Drafted rows on the device (q3h_cache_*, q3h_rope_*, q3h_token_logprobs)
against float64, through the binding's tensors."""
import gc

import numpy as np
import pytest
import torch

import draft_ref as ref
import q3h

pytestmark = pytest.mark.gpu

F, H, Q = q3h.KV_F32, q3h.KV_F16, q3h.KV_Q8
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def no_handles_left():
    """Handles that a refusal's traceback still holds go before the device does."""
    yield
    gc.collect()


def dev_i(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def dev_f(v):
    return torch.tensor(np.asarray(v, np.float32), device="cuda")


def host(t):
    return t.detach().float().cpu().numpy()


def random_tree(rng, n, rows):
    back = rng.geometric(0.4, (n, rows))
    return np.maximum(np.arange(rows)[None] - back, -1).astype(np.int32)


def fill(cache, k, v, held):
    """Positions [0, held[b]) of every sequence from f32 rows [n][rows][kvh][hd]."""
    n = k.shape[0]
    if k.shape[1]:
        cache.append(dev_f(k), dev_f(v), dev_i([0] * n), counts=dev_i(held))


ROPES = {
    "plain": dict(),
    "half_of_head": dict(rot=0.5, scaling=dict(kind="linear", factor=2.0)),
    "pairs": dict(interleaved=True),
    "pairs_of_six": dict(rot=6, interleaved=True, scaling=dict(kind="bands", factor=8.0,
                                                             original=512)),
    "yarn": dict(scaling=dict(kind="yarn", factor=4.0, original=1024)),
    "halves_of_ten": dict(rot=20, scaling=dict(kind="linear", factor=3.0)),
    "none": None,
}


@pytest.mark.parametrize("fmt", [F, H, Q])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rope", list(ROPES))
@pytest.mark.parametrize("tree", [False, True])
def test_append_rounds_the_definition(device, fmt, hd, rope, tree):
    """Normed, turned and stored rows: q within half a step of f32, what the
    cache holds equal to the format of the f32 row."""
    print(f"append fmt {fmt} hd {hd} rope {rope} tree {tree}", flush=True)
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
    cache = q3h.Cache(device, n, kvh, hd, P, fmt, layers=2)
    qkv = rng.standard_normal((n, rows, (heads + 2 * kvh) * hd + 8)).astype(np.float32)
    qkv *= np.exp(rng.standard_normal((n, rows, 1))).astype(np.float32)
    norm = r is not None and rope != "pairs"
    qn = (1 + 0.2 * rng.standard_normal(hd)).astype(np.float32)
    kn = (1 + 0.2 * rng.standard_normal(hd)).astype(np.float32)
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
    other = torch.full((n, P, kvh, hd), 7.0, device="cuda")
    cache.read(other, None, layer=0)
    assert not other.any()  # the other layer is untouched
    held = torch.zeros((n, P, kvh, hd), device="cuda")
    cache.read(held, None, layer=1)
    for s in range(n):
        inside = np.zeros(P, bool)
        inside[lens[s]:lens[s] + counts[s]] = True
        assert not host(held[s])[~inside].any()
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
            np.testing.assert_array_equal(k[s, i], ref.stored(k0.astype(np.float32), fmt))
            v0 = qkv[s, i, b:b + kvh * hd].reshape(kvh, hd)
            np.testing.assert_array_equal(v[s, i], ref.stored(v0, fmt))


def test_append_in_place_and_without_queries(device):
    rng = np.random.default_rng(3)
    cache = q3h.Cache(device, 2, 2, 128, 64, F)
    table = q3h.Rope(device, 128, 64, 1e4)
    x = dev_f(rng.standard_normal((2, 5, 8, 128)))
    k = dev_f(rng.standard_normal((2, 5, 2, 128)))
    lens = dev_i([3, 50])
    want = cache.append(k, k, lens, q=x, rope=table).clone()
    y = x.clone()
    assert cache.append(k, k, lens, q=y, q_out=y, rope=table) is y
    assert torch.equal(y, want)
    assert cache.append(k, k, lens, rope=table) is None


@pytest.mark.parametrize("fmt", [F, H, Q])
def test_rows_of_extreme_values(device, fmt):
    """Zeros, the smallest and largest values, infinities and NaN, a row each."""
    hd = 64
    rng = np.random.default_rng(5)
    x = rng.standard_normal((9, hd)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e-44)
    x[2] *= np.float32(3e-39)
    x[3] = np.float32(3.3e38) * np.sign(x[3])
    x[4, 5] = np.inf
    x[5, 63] = -np.inf
    x[6, 0] = np.nan
    x[7] *= np.float32(6e4)
    x[8, :] = 0
    x[8, 9] = np.float32(1e-45)
    cache = q3h.Cache(device, 1, 1, hd, 16, fmt)
    rows = dev_f(x[None, :, None])
    cache.append(rows, rows, dev_i([0]))
    k, v = torch.zeros_like(rows), torch.zeros_like(rows)
    cache.read(k, v)
    want = ref.stored(x, fmt)
    np.testing.assert_array_equal(host(k)[0, :, 0], want)
    np.testing.assert_array_equal(host(v)[0, :, 0], want)


def test_bad_lengths_and_parents_write_nothing(device):
    """A sequence out of range or a broken path: NaN queries, no row in the
    cache; the sequences beside it as ever."""
    rng = np.random.default_rng(9)
    n, rows, P = 5, 4, 16
    cache = q3h.Cache(device, n, 2, 64, P, Q)
    q = dev_f(rng.standard_normal((n, rows, 2, 64)))
    k = dev_f(rng.standard_normal((n, rows, 2, 64)))
    lens = dev_i([2, 13, -1, 2 ** 31 - 2, 5])
    parents = np.tile(np.arange(rows) - 1, (n, 1)).astype(np.int32)
    parents[4] = [-1, 0, 2, 1]  # row 2 is its own parent; row 3 does not meet it
    out = host(cache.append(k, k, lens, q=q, parents=dev_i(parents)))
    everything = torch.zeros((n, P, 2, 64), device="cuda")
    cache.read(everything, None)
    e = host(everything)
    assert np.isfinite(out[0]).all() and (np.abs(e[0, 2:6]).max(-1) > 0).all()
    for s in (1, 2, 3):
        assert np.isnan(out[s]).all() and not e[s].any()
    assert np.isnan(out[4, 2]).all() and np.isfinite(out[4, [0, 1, 3]]).all()
    assert not e[4, 7].any() and (np.abs(e[4, [5, 6, 8]]).max(-1) > 0).all()
    # the same lengths read and attended: NaN, nothing out of range
    r = torch.zeros((n, rows, 2, 64), device="cuda")
    cache.read(r, None, starts=lens)
    assert np.isnan(host(r)[1:4]).all() and np.isfinite(host(r)[0]).all()
    o = host(cache.attend(q, lens, 12, parents=dev_i(parents)))
    assert np.isfinite(o[0]).all() and np.isnan(o[1:4]).all()
    assert np.isnan(o[4, 2]).all() and np.isfinite(o[4, [0, 1, 3]]).all()
    # a length above max_len
    o = host(cache.attend(q, dev_i([2, 0, 0, 0, 5]), 4, parents=dev_i(parents)))
    assert np.isfinite(o[0]).all() and np.isnan(o[4]).all()


ATTEND = [
    # (fmt, hd, heads, kv_heads, rows, lens, tree)
    (F, 128, 16, 8, 1, [0], False),
    (F, 128, 16, 8, 1, [1, 200, 31], False),
    (H, 128, 16, 8, 1, [63, 64, 65], False),
    (Q, 128, 4, 2, 1, [0, 32, 33, 500], False),
    (F, 64, 6, 2, 5, [7, 0, 90], True),
    (H, 64, 4, 4, 17, [15, 1000], True),
    (Q, 64, 8, 1, 64, [33, 2], True),
    (F, 128, 4, 2, 64, [100], True),
    (H, 128, 28, 4, 11, [1, 95, 350], True),
    (Q, 128, 16, 4, 33, [127, 640], True),
    (F, 128, 2, 1, 100, [40, 0], False),
    (H, 64, 3, 1, 129, [5, 77], False),
    (Q, 128, 8, 2, 70, [300, 1], False),
    (Q, 128, 2, 1, 1, [4100, 2000], False),
    (H, 128, 2, 1, 9, [4500], True),
    (F, 64, 2, 1, 2, [3333, 4097], False),
    (H, 64, 8, 2, 300, [900, 350, 0], False),
    (Q, 128, 8, 8, 2, [900 - 13 * i for i in range(50)], True),
    (H, 128, 4, 1, 64, [2000, 100, 1500, 30], True),
]


@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attend_matches_float64(device, case):
    fmt, hd, heads, kvh, rows, lens, tree = ATTEND[case]
    print("attend", ATTEND[case], flush=True)
    rng = np.random.default_rng(100 + case)
    n, P = len(lens), max(lens) + rows + 3
    lens = np.array(lens)
    counts = np.array([max(1, rows - i * 3) for i in range(n)])
    k = rng.standard_normal((n, P, kvh, hd)).astype(np.float32) * \
        np.exp(0.5 * rng.standard_normal((kvh, hd))).astype(np.float32)
    v = rng.standard_normal((n, P, kvh, hd)).astype(np.float32)
    q = rng.standard_normal((n, rows, heads, hd)).astype(np.float32) * 2
    parents = random_tree(rng, n, rows) if tree else None
    cache = q3h.Cache(device, n, kvh, hd, P, fmt)
    fill(cache, k, v, lens + counts)
    wide = np.zeros((n, rows, heads * hd + 12), np.float32)  # rows further apart
    wide[..., :heads * hd] = q.reshape(n, rows, -1)
    out = torch.full((n, rows, heads, hd), 7.0, device="cuda")
    cache.attend(dev_f(wide)[..., :heads * hd], dev_i(lens), int(lens.max()), out=out,
                 counts=dev_i(counts), parents=None if parents is None else dev_i(parents))
    held = ref.stored(k, fmt).astype(np.float64), ref.stored(v, fmt).astype(np.float64)
    want, bound = ref.attention(q.astype(np.float64), *held, lens, counts, parents, hd ** -0.5)
    out = host(out)
    for s in range(n):
        assert (out[s, counts[s]:] == 7).all()
        d = np.abs(out[s, :counts[s]] - want[s, :counts[s]])
        worst = float((d / np.maximum(bound[s, :counts[s]], 1e-300)).max())
        print(f"sequence {s}: {d.max():.2e}, {worst:.2e} of the bound", flush=True)
        assert worst <= 1
    # in place, with a longer bound and a scale of its own: the same rows
    x = dev_f(q)
    got = cache.attend(x, dev_i(lens), P, out=x, counts=dev_i(counts), scale=hd ** -0.5,
                       parents=None if parents is None else dev_i(parents))
    got = host(got)
    for s in range(n):
        d = np.abs(got[s, :counts[s]] - want[s, :counts[s]])
        assert (d <= bound[s, :counts[s]]).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kvh,rows", [(4, 2, 1), (3, 3, 1), (3, 3, 2)])
@pytest.mark.parametrize("tree", [False, True])
def test_attend_of_one_or_two_rows(device, hd, heads, kvh, rows, tree):
    """Single tokens and pairs over short f32 caches, with infinities and NaN where
    a row does not look, counts of none, bad parents and lengths."""
    rng = np.random.default_rng(37)
    lens = np.array([0, 1, 15, 16, 17, 95, 96, 97, 171, 300, 301, 40, 33, 8])
    n, P = len(lens), 310
    counts = np.array([rows] * n)
    counts[4], counts[5] = 0, 1
    parents = np.array([[-1, -1 + (i % 2)][:rows] for i in range(n)], np.int32)
    if tree and rows == 2:
        parents[11], parents[12] = [-1, 1], [0, 0]
    if tree and rows == 1:
        parents[11], parents[12] = [0], [-2]
    k, v = [rng.standard_normal((n, P, kvh, hd)).astype(np.float32) for _ in range(2)]
    for b in range(n):
        k[b, lens[b] + rows:, :, 3] = np.nan
        v[b, lens[b] + rows:, :, 5] = np.inf
        if tree and rows == 2 and parents[b, 1] == -1:  # row 1 does not see row 0
            k[b, lens[b]], v[b, lens[b]] = np.nan, -np.inf
    q = (2 * rng.standard_normal((n, rows, heads, hd))).astype(np.float32)
    cache = q3h.Cache(device, n, kvh, hd, P, F)
    fill(cache, k, v, [P] * n)
    asked = lens.copy()
    asked[13] = -3
    out = torch.full((n, rows, heads, hd), 7.0, device="cuda")
    cache.attend(dev_f(q), dev_i(asked), 302, out=out, counts=dev_i(counts),
                 parents=dev_i(parents) if tree else None)
    same = dev_f(q)  # in place
    cache.attend(same, dev_i(asked), 302, out=same, counts=dev_i(counts),
                 parents=dev_i(parents) if tree else None)
    out, same = host(out), host(same)
    assert np.isnan(out[13]).all()
    for b in range(13):
        assert (out[b, counts[b]:] == 7).all() and (same[b, counts[b]:] == q[b, counts[b]:]).all()
        for t in range(counts[b]):
            np.testing.assert_array_equal(out[b, t], same[b, t])
            if tree and (b == 12 or (b == 11 and t == rows - 1)):
                assert np.isnan(out[b, t]).all()
                continue
            if tree and rows == 2 and t == 0 and parents[b, 1] == -1:
                assert np.isnan(out[b, t]).all()  # it sees its own NaN
                continue
            want, bound = ref.attention(
                q[b:b + 1].astype(np.float64), k[b:b + 1].astype(np.float64),
                v[b:b + 1].astype(np.float64), [lens[b]], [t + 1],
                parents[b:b + 1] if tree else None, hd ** -0.5)
            assert (np.abs(out[b, t] - want[0, t]) <= bound[0, t]).all()


@pytest.mark.parametrize("fmt", [F, H, Q])
@pytest.mark.parametrize("heads", [2, 32])
def test_unseen_rows_do_not_reach_a_row(device, fmt, heads):
    """Infinities and NaN in siblings' and in stale positions."""
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
    cache = q3h.Cache(device, 1, 2, hd, P, fmt)
    fill(cache, k, v, [P])
    out = host(cache.attend(dev_f(q), dev_i([length]), length, parents=dev_i(parents)))
    clean = [0, 1, 3, 5, 7, 8, 9, 10, 11]
    assert np.isnan(out[0, [2, 4, 6]]).all()
    kk, vv = np.nan_to_num(ref.stored(k, fmt), nan=0, posinf=0, neginf=0), \
        np.nan_to_num(ref.stored(v, fmt), nan=0, posinf=0, neginf=0)
    want, bound = ref.attention(q.astype(np.float64), kk.astype(np.float64), vv.astype(np.float64),
                                [length], [rows], parents, hd ** -0.5)
    assert (np.abs(out - want)[0, clean] <= bound[0, clean]).all()
    # a chain sees all that came before it
    out = host(cache.attend(dev_f(q), dev_i([length]), length))
    assert np.isfinite(out[0, :2]).all() and np.isnan(out[0, 2:]).all()


@pytest.mark.parametrize("fmt", [F, H, Q])
@pytest.mark.parametrize("heads", [2, 24])
def test_large_values_of_siblings_cost_no_precision(device, fmt, heads):
    """Siblings whose values are larger by up to 2^100, and positions before the
    draft whose values are smaller by 2^30, leave a row's precision as it is."""
    rng = np.random.default_rng(24)
    hd, rows, P, length = 64, 7, 200, 150
    k = rng.standard_normal((1, P, 1, hd)).astype(np.float32)
    v = rng.standard_normal((1, P, 1, hd)).astype(np.float32)
    v[0, :100] *= 2.0 ** (-10 if fmt == H else -30)
    parents = np.array([[-1, -1, 0, 1, 2, 3, 4]], np.int32)
    for r in (1, 3, 5):  # a branch of its own
        v[0, length + r] *= 2.0 ** (12 if fmt == H else 33 * (r + 1) // 2)
    k[0, length:] *= 0.1
    q = rng.standard_normal((1, rows, heads, hd)).astype(np.float32)
    cache = q3h.Cache(device, 1, 1, hd, P, fmt)
    fill(cache, k, v, [length + rows])
    out = host(cache.attend(dev_f(q), dev_i([length]), length, parents=dev_i(parents)))
    held = ref.stored(k, fmt).astype(np.float64), ref.stored(v, fmt).astype(np.float64)
    want, bound = ref.attention(q.astype(np.float64), *held, [length], [rows], parents, hd ** -0.5)
    assert np.isfinite(want).all()
    ratio = np.abs(out - want) / bound
    print(ratio.max(axis=(0, 2, 3)), flush=True)
    assert (ratio <= 1).all()


@pytest.mark.parametrize("size", [2.0 ** -110, 2.0 ** -70, 2.0 ** -50, 2.0 ** 45, 2.0 ** 70, 2.0 ** 110])
@pytest.mark.parametrize("heads", [1, 20])
def test_attend_int8_values_of_any_size(device, size, heads):
    rng = np.random.default_rng(26)
    hd, rows, P, length = 128, 3, 300, 290
    k = rng.standard_normal((1, P, 1, hd)).astype(np.float32)
    v = (rng.standard_normal((1, P, 1, hd)) * size).astype(np.float32)
    v[0, 64:96] = 0
    v[0, 200:240] *= 2.0 ** -16
    q = rng.standard_normal((1, rows, heads, hd)).astype(np.float32)
    cache = q3h.Cache(device, 1, 1, hd, P, Q)
    fill(cache, k, v, [length + rows])
    held = ref.stored(k, Q).astype(np.float64), ref.stored(v, Q).astype(np.float64)
    want, bound = ref.attention(q.astype(np.float64), *held, [length], [rows], None, hd ** -0.5)
    out = host(cache.attend(dev_f(q), dev_i([length]), length))
    ratio = np.abs(out - want) / bound
    print(ratio.max(), flush=True)
    assert (ratio <= 1).all()


@pytest.mark.parametrize("fmt", [F, H, Q])
def test_attend_with_other_scales(device, fmt):
    """A scale so small that every position counts the same, one that takes the
    queries' products out of f32's normal numbers, a negative one."""
    rng = np.random.default_rng(25)
    hd, rows, P, length = 128, 5, 90, 61
    k = rng.standard_normal((2, P, 2, hd)).astype(np.float32)
    v = rng.standard_normal((2, P, 2, hd)).astype(np.float32)
    q = rng.standard_normal((2, rows, 4, hd)).astype(np.float32)
    parents = random_tree(rng, 2, rows)
    cache = q3h.Cache(device, 2, 2, hd, P, fmt)
    fill(cache, k, v, [P, P])
    held = ref.stored(k, fmt).astype(np.float64), ref.stored(v, fmt).astype(np.float64)
    for scale in (1e-20, 1e-40, -0.11):
        want, bound = ref.attention(q.astype(np.float64), *held, [length, 3], [rows] * 2, parents,
                                    scale)
        out = host(cache.attend(dev_f(q), dev_i([length, 3]), length, parents=dev_i(parents),
                                scale=scale))
        assert (np.abs(out - want) <= bound).all()


def test_infinite_values_seen_stay_infinite(device):
    """An infinity among the values a row sees comes out in its element, as in
    the sum that defines it, and in no other."""
    rng = np.random.default_rng(22)
    hd, rows, length = 64, 3, 20
    for fmt in (F, H):
        k = rng.standard_normal((1, 40, 1, hd)).astype(np.float32)
        v = rng.standard_normal((1, 40, 1, hd)).astype(np.float32)
        v[0, 4, 0, 10] = np.inf
        v[0, length + 1, 0, 11] = -np.inf
        cache = q3h.Cache(device, 1, 1, hd, 40, fmt)
        fill(cache, k, v, [length + rows])
        q = rng.standard_normal((1, rows, 2, hd)).astype(np.float32)
        out = host(cache.attend(dev_f(q), dev_i([length]), length,
                                parents=dev_i([[-1, 0, 0]])))[0]
        assert (out[:, :, 10] == np.inf).all()
        assert (out[1, :, 11] == -np.inf).all() and np.isfinite(out[[0, 2]][:, :, 11]).all()
        rest = [e for e in range(hd) if e not in (10, 11)]
        assert np.isfinite(out[:, :, rest]).all()


def test_large_and_small_scores(device):
    """Scores far apart and large: the softmax's maximum is its own row's."""
    rng = np.random.default_rng(23)
    hd, rows, length = 128, 5, 300
    k = rng.standard_normal((1, 400, 2, hd)).astype(np.float32) * 30
    v = rng.standard_normal((1, 400, 2, hd)).astype(np.float32) * 1000
    q = rng.standard_normal((1, rows, 4, hd)).astype(np.float32)
    q[0, 0] *= 1e-30
    q[0, 1] *= 100
    q[0, 2] *= 1e4
    q[0, 3] = 0
    for fmt in (F, H, Q):
        cache = q3h.Cache(device, 1, 2, hd, 400, fmt)
        fill(cache, k, v, [length + rows])
        out = host(cache.attend(dev_f(q), dev_i([length]), length))
        want, bound = ref.attention(q.astype(np.float64), ref.stored(k, fmt).astype(np.float64),
                                    ref.stored(v, fmt).astype(np.float64), [length], [rows], None,
                                    hd ** -0.5)
        assert (np.abs(out - want) <= bound).all()


def test_offsets_past_32_bits(device):
    """Two million positions of 8 heads: elements and bytes past 2^31."""
    hd, kvh, P = 128, 8, (1 << 21) + 40
    length = (1 << 21) + 9
    rng = np.random.default_rng(31)
    cache = q3h.Cache(device, 1, kvh, hd, P, Q)
    k = rng.standard_normal((1, 2, kvh, hd)).astype(np.float32)
    v = rng.standard_normal((1, 2, kvh, hd)).astype(np.float32) * 1e5
    q = rng.standard_normal((1, 2, kvh, hd)).astype(np.float32) * 3
    cache.append(dev_f(k), dev_f(v), dev_i([length]))
    back_k, back_v = torch.zeros((1, 2, kvh, hd), device="cuda"), \
        torch.zeros((1, 2, kvh, hd), device="cuda")
    cache.read(back_k, back_v, starts=dev_i([length]))
    np.testing.assert_array_equal(host(back_k), ref.stored(k, Q))
    np.testing.assert_array_equal(host(back_v), ref.stored(v, Q))
    out = host(cache.attend(dev_f(q), dev_i([length]), length))
    kk, vv = ref.stored(k, Q).astype(np.float64), ref.stored(v, Q).astype(np.float64)
    for t in range(2):  # the positions before are zeros: weight e^0 each
        for a in range(kvh):
            s = kk[0, :t + 1, a] @ q[0, t, a].astype(np.float64) * hd ** -0.5
            w = np.exp(s)
            want = w @ vv[0, :t + 1, a] / (length + w.sum())
            # sums of 2^21 equal terms, over a thousand in a row at most
            np.testing.assert_allclose(out[0, t, a], want, rtol=2e-4,
                                       atol=2e-4 * np.abs(want).max())


@pytest.mark.parametrize("fmt", [F, H, Q])
@pytest.mark.parametrize("hd", [64, 128])
def test_keep_moves_the_path_forward(device, fmt, hd):
    rng = np.random.default_rng(41)
    n, rows, P, layers = 4, 7, 40, 2
    cache = q3h.Cache(device, n, 2, hd, P, fmt, layers=layers)
    lens = np.array([3, 0, 33, 20])
    x = rng.standard_normal((layers, 2, n, P, 2, hd)).astype(np.float32)
    for l in range(layers):
        cache.append(dev_f(x[l, 0]), dev_f(x[l, 1]), dev_i([0] * n), layer=l)
    kept = np.array([[0, 2, 5, 9, 9, 9, 9], [6, 0, 0, 0, 0, 0, 0], [0, 1, 2, 3, 4, 5, 6],
                     [1, 1, 2, 0, 0, 0, 0]])
    counts = np.array([3, 1, 7, 2])  # the last list repeats a row: left alone
    cache.keep(dev_i(lens), dev_i(kept), dev_i(counts))
    for l in range(layers):
        k, v = (torch.zeros((n, P, 2, hd), device="cuda") for _ in range(2))
        cache.read(k, v, layer=l)
        for part, got in ((0, host(k)), (1, host(v))):
            want = ref.stored(x[l, part], fmt)
            for b in range(3):
                for i in range(counts[b]):
                    want[b, lens[b] + i] = ref.stored(x[l, part, b, lens[b] + kept[b, i]], fmt)
            np.testing.assert_array_equal(got, want)


SCORES = [
    # (rows, vocab, dtype, tokens, top_k)
    (1, 1, "float32", 1, 1), (3, 5, "float32", 2, 5), (7, 64, "bfloat16", 1, 64),
    (2, 100, "float32", 3, 0), (5, 2048, "float32", 1, 10), (1, 151936, "float32", 4, 64),
    (3, 40001, "bfloat16", 1, 33), (300, 1031, "bfloat16", 2, 3), (1100, 257, "float32", 1, 1),
    (40, 8192, "float32", 1, 20),
]


def check_scores(got, x, tokens, top_k):
    logprobs, entropy, ids, top = ref.scores(x, tokens, top_k)
    vocab = x.shape[1]
    finite = np.where(np.isfinite(x), np.abs(x), 0).max(-1)
    # the sum of the exponentials: at most vocab / 64 terms in a row, each within
    # 2^-22; then a logarithm and two differences of numbers up to the logits'
    rel = (vocab / 64 + 32) * U
    tol = (rel + 4 * U * (1 + 2 * finite))[:, None]
    for name, want in (("logprobs", logprobs), ("top_logprobs", top)):
        if want.size == 0:
            continue
        g = host(got[name])
        np.testing.assert_array_equal(np.isnan(g), np.isnan(want))
        np.testing.assert_array_equal(np.isinf(g), np.isinf(want))
        with np.errstate(invalid="ignore"):
            d = np.abs(g - want)
        assert (np.where(np.isfinite(want), d, 0) <= tol).all()
    g = host(got["entropy"])
    np.testing.assert_array_equal(np.isnan(g), np.isnan(entropy))
    d = np.where(np.isnan(entropy), 0, np.abs(g - entropy))
    assert (d <= tol[:, 0] * (2 + np.log(vocab))).all()
    if top_k:
        np.testing.assert_array_equal(got["top_ids"].cpu().numpy(), ids)


@pytest.mark.parametrize("case", range(len(SCORES)))
def test_scores_match_float64(device, case):
    rows, vocab, dtype, m, top_k = SCORES[case]
    print("scores", SCORES[case], flush=True)
    rng = np.random.default_rng(200 + case)
    x = dev_f(rng.standard_normal((rows, vocab)) * 3).to(getattr(torch, dtype))
    wide = torch.full((rows, vocab + 5), float("nan"), device="cuda", dtype=x.dtype)
    wide[:, :vocab] = x
    tokens = rng.integers(0, vocab, (rows, m)).astype(np.int32)
    if m > 1:
        tokens[0, 0], tokens[-1, 1] = -1, vocab
    got = q3h.token_logprobs(device, wide[:, :vocab], dev_i(tokens), top_k=top_k)
    assert ("top_ids" in got) == (top_k > 0)
    check_scores(got, host(x), tokens, top_k)


def test_scores_of_ties_and_strange_rows(device):
    rng = np.random.default_rng(61)
    vocab = 3000
    x = rng.integers(-2, 3, (14, vocab)).astype(np.float32)  # ties everywhere
    x[1] = 0.5
    x[2] = -np.inf
    x[3, :] = -np.inf
    x[3, 2999] = 1e30
    x[4, 17] = np.inf
    x[5, 40] = np.nan
    x[6] = np.nan
    x[7, ::2] = -np.inf
    x[8] = -3.4e38
    x[9] = 3.4e38
    x[10, :2990] = -np.inf
    x[11, 5:] = np.nan
    x[12] = -0.0
    x[12, 1000:] = 0.0
    tokens = np.tile(np.array([[0, 2999, 17]], np.int32), (14, 1))
    for top_k in (1, 20, 64):
        got = q3h.token_logprobs(device, dev_f(x), dev_i(tokens), top_k=top_k)
        check_scores(got, x, tokens, top_k)


def test_a_drafted_step(device):
    """The operators as they are used: prompts, a drafted tree, its scores, the
    kept path, the next tree; every row's attention as float64 gives it from
    the rows themselves."""
    rng = np.random.default_rng(71)
    n, heads, kvh, hd, rows, P, vocab = 3, 4, 2, 64, 9, 160, 500
    lens = np.array([40, 0, 71])
    freq, mag = ref.frequencies(hd, 1e4)
    for fmt in (F, H, Q):
        cache = q3h.Cache(device, n, kvh, hd, P, fmt)
        table = q3h.Rope(device, hd, P, 1e4)
        held = [[], [], []]  # the turned keys and the values of each sequence

        def rows_of(count):
            return (rng.standard_normal((n, count, heads, hd)).astype(np.float32),
                    rng.standard_normal((n, count, kvh, hd)).astype(np.float32),
                    rng.standard_normal((n, count, kvh, hd)).astype(np.float32))

        def keys(k, pos):
            y = ref.turned(k.astype(np.float64), pos, hd, False, freq, mag)
            return ref.stored(y.astype(np.float32), fmt).astype(np.float64)

        q, k, v = rows_of(71)
        cache.append(dev_f(k), dev_f(v), dev_i([0] * n), counts=dev_i(lens), rope=table)
        for b in range(n):
            held[b] = [(keys(k[b, i], i), ref.stored(v[b, i], fmt).astype(np.float64))
                       for i in range(lens[b])]
        now = lens.copy()
        head = rng.standard_normal((heads * hd, vocab)).astype(np.float32) * 0.3
        for step in range(3):
            q, k, v = rows_of(rows)
            parents = random_tree(rng, n, rows)
            qt = cache.append(dev_f(k), dev_f(v), dev_i(now), parents=dev_i(parents), q=dev_f(q),
                              rope=table)
            out = cache.attend(qt, dev_i(now), int(now.max()), parents=dev_i(parents))
            logits = out.reshape(n * rows, heads * hd) @ dev_f(head)
            tokens = rng.integers(0, vocab, (n * rows, 2)).astype(np.int32)
            got = q3h.token_logprobs(device, logits, dev_i(tokens), top_k=4)
            check_scores(got, host(logits), tokens, 4)
            out = host(out)
            kept, kept_n = np.zeros((n, rows), np.int32), []
            for b in range(n):
                kk = np.zeros((1, now[b] + rows, kvh, hd))
                vv, qq = np.zeros_like(kk), np.zeros((1, rows, heads, hd))
                for i, (a, c) in enumerate(held[b]):
                    kk[0, i], vv[0, i] = a, c
                for t in range(rows):
                    pos = now[b] + len(ref.path(parents[b], t)) - 1
                    kk[0, now[b] + t] = keys(k[b, t], pos)
                    vv[0, now[b] + t] = ref.stored(v[b, t], fmt)
                    qq[0, t] = ref.turned(q[b, t].astype(np.float64), pos, hd, False, freq, mag)
                want, bound = ref.attention(qq, kk, vv, [now[b]], [rows], parents[b:b + 1],
                                            hd ** -0.5)
                # (the queries are rounded to f32 once: within the bound's terms)
                assert (np.abs(out[b] - want[0]) <= bound[0]).all()
                p = ref.path(parents[b], int(rng.integers(rows)))[::-1]
                kept[b, :len(p)] = p
                kept_n.append(len(p))
                held[b] += [(kk[0, now[b] + t], vv[0, now[b] + t]) for t in p]
            cache.keep(dev_i(now), dev_i(kept), dev_i(kept_n))
            now = now + np.array(kept_n)
        k2, v2 = (torch.zeros((n, P, kvh, hd), device="cuda") for _ in range(2))
        cache.read(k2, v2, counts=dev_i(now))
        for b in range(n):
            np.testing.assert_array_equal(host(k2)[b, :now[b]], np.array([a for a, _ in held[b]]))
            np.testing.assert_array_equal(host(v2)[b, :now[b]], np.array([c for _, c in held[b]]))


def test_captured_calls_follow_lengths_on_the_device(device):
    """One graph of append, attention and scores, replayed as the lengths grow;
    another over the same cache with a workspace of its own beside it; eager
    calls in between."""
    rng = np.random.default_rng(81)
    n, heads, kvh, hd, P, vocab = 2, 8, 2, 128, 3000, 700
    cache = q3h.Cache(device, n, kvh, hd, P, Q)
    table = q3h.Rope(device, hd, P, 1e6)
    base = rng.standard_normal((n, 2200, kvh, hd)).astype(np.float32)
    fill(cache, base, base, [2200, 1500])
    head = dev_f(rng.standard_normal((heads * hd, vocab)) * 0.1)
    lens = dev_i([2200, 1500])
    q, k, v = (dev_f(rng.standard_normal((n, 4, h, hd))) for h in (heads, kvh, kvh))
    parents = dev_i([[-1, 0, 0, 1]] * n)
    tokens = dev_i(rng.integers(0, vocab, (4 * n, 1)))

    def step(space=None):
        qt = cache.append(k, v, lens, parents=parents, q=q, rope=table)
        out = cache.attend(qt, lens, 2900, parents=parents, workspace=space)
        s = q3h.token_logprobs(device, out.reshape(4 * n, -1) @ head, tokens, top_k=3)
        return out, s["logprobs"], s["top_ids"]

    need = max(1, cache.attend_workspace(n, 4, heads, 2900))
    graphs = []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()  # (library workspaces of the product before any capture)
    torch.cuda.synchronize()
    for _ in range(2):
        space = torch.empty(need, dtype=torch.uint8, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(space)
        graphs.append((g, res, space))
    for i in range(4):
        q.copy_(dev_f(rng.standard_normal((n, 4, heads, hd))))
        k.copy_(dev_f(rng.standard_normal((n, 4, kvh, hd))))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for g, res, _ in graphs:
            for t in res:
                t.zero_()
            g.replay()
        torch.cuda.synchronize()
        for _, res, _ in graphs:
            for a, b in zip(res, want):
                assert torch.equal(a, b)
        lens += 3


def test_calls_on_another_stream(device):
    """Work queued on a stream of the caller's is seen by calls on it."""
    cache = q3h.Cache(device, 1, 2, 64, 600, H)
    rng = np.random.default_rng(91)
    k = dev_f(rng.standard_normal((1, 512, 2, 64)))
    q = dev_f(rng.standard_normal((1, 1, 4, 64)))
    lens = dev_i([511])
    cache.append(k, k, dev_i([0]))
    want = cache.attend(q, lens, 511).clone()
    cache.append(torch.zeros_like(k), torch.zeros_like(k), dev_i([0]))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    late = torch.zeros_like(k)
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(4):
            big = big @ big
            big /= big.norm()
        late.copy_(k)
        cache.append(late, late, dev_i([0]))
        got = cache.attend(q, lens, 511)
    s.synchronize()
    assert torch.equal(got, want)
    assert torch.cuda.current_device() == 0


def test_empty_calls(device):
    cache = q3h.Cache(device, 2, 2, 64, 8, F)
    none = torch.zeros((0, 3, 2, 64), device="cuda")
    i0 = torch.zeros(0, dtype=torch.int32, device="cuda")
    cache.append(none, none, i0)
    assert cache.attend(none, i0, 8).shape == (0, 3, 2, 64)
    zero_rows = torch.zeros((2, 0, 2, 64), device="cuda")
    cache.append(zero_rows, zero_rows, dev_i([8, 8]))
    assert cache.attend(zero_rows, dev_i([8, 8]), 8).shape == (2, 0, 2, 64)
    cache.read(zero_rows, None)
    s = q3h.token_logprobs(device, torch.zeros((0, 9), device="cuda"),
                           torch.zeros((0, 1), dtype=torch.int32, device="cuda"), top_k=2)
    assert s["logprobs"].shape == (0, 1) and s["top_ids"].shape == (0, 2)


def test_refusals_of_tensors(device):
    cache = q3h.Cache(device, 2, 2, 64, 8, F)
    k = torch.zeros((2, 3, 2, 64), device="cuda")
    lens = dev_i([0, 0])
    bad = [
        lambda: cache.append(k.cpu(), k, lens),
        lambda: cache.append(k.half(), k, lens),
        lambda: cache.append(k, k, lens.long()),
        lambda: cache.append(k, k, dev_i([0, 0, 0])),
        lambda: cache.append(k, k[:, :, :1], lens),
        lambda: cache.append(k.transpose(2, 3), k, lens),
        lambda: cache.append(k[:, ::2], k[:, :2], lens),
        lambda: cache.attend(torch.zeros((2, 3, 3, 64), device="cuda"), lens, 8),
        lambda: cache.attend(k, lens, 9),
        lambda: cache.attend(k, lens, 8, scale=float("nan")),
        lambda: cache.read(k.transpose(0, 1), None),
        lambda: q3h.Cache(device, 2, 2, 96, 8, F),
        lambda: q3h.Rope(device, 64, 8, 1e4, rot_dim=7),
        lambda: q3h.Rope(device, 64, 8, 1e4, scaling=dict(kind="yarn", factor=2.0)),
        lambda: q3h.token_logprobs(device, k[0, 0], dev_i([[0], [0]]), top_k=65),
        lambda: q3h.token_logprobs(device, k[0, 0].half(), dev_i([[0], [0]])),
    ]
    for f in bad:
        with pytest.raises(q3h.Q3HError) as e:
            f()
        assert e.value.code == q3h.E_ARG
    with pytest.raises(q3h.Q3HError) as e:
        wide = torch.zeros((1, 70, 2, 64), device="cuda")
        q3h.Cache(device, 1, 2, 64, 100, F).append(wide, wide, dev_i([0]),
                                                   parents=dev_i([[-1] * 70]))
    assert e.value.code == q3h.E_CAPACITY
    table = q3h.Rope(device, 64, 4, 1e4)
    with pytest.raises(q3h.Q3HError):
        cache.append(k, k, lens, rope=table)  # fewer positions than the cache


def test_destroyed_handles_are_refused(device):
    """A destroyed table is not taken for none, a destroyed cache for any."""
    cache = q3h.Cache(device, 1, 1, 64, 16)
    table = q3h.Rope(device, 64, 16, 1e4)
    rows, lens = torch.ones(1, 2, 1, 64, device="cuda"), dev_i([0])
    cache.append(rows, rows, lens, rope=table)
    table.destroy()
    with pytest.raises(Exception, match="destroyed"):
        cache.append(rows, rows, lens, rope=table)
    with pytest.raises(Exception, match="neither"):
        cache.read(None, None)
    cache.destroy()
    for call in (lambda: cache.append(rows, rows, lens), lambda: cache.attend(rows, lens, 0),
                 lambda: cache.read(rows, None)):
        with pytest.raises(q3h.Q3HError):
            call()


@pytest.mark.parametrize("fmt", [F, H, Q])
@pytest.mark.parametrize("hd", [64, 128])
def test_append_of_any_heads_and_distances(device, fmt, hd):
    """Heads that fill a wave, part of one and several, none of the queries',
    rows that begin between 16-byte boundaries."""
    rng = np.random.default_rng(33 + hd + fmt)
    freq, mag = ref.frequencies(hd, 1e4)
    table = q3h.Rope(device, hd, 50, 1e4)
    qn, kn = [(1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    eps = float(np.float32(1e-6))

    def place(x, ld):  # rows ld floats apart, from an odd float on
        n, rows = x.shape[:2]
        buf = torch.full((n * rows * ld + 1,), 9.0, device="cuda")
        t = buf[1:].as_strided((n, rows, x.shape[2] * hd), (rows * ld, ld, 1), 1)
        t.copy_(dev_f(x).reshape(n, rows, -1))
        return t

    for heads, kvh in ((0, 1), (1, 1), (5, 1), (28, 4), (7, 7), (48, 8), (12, 9)):
        print("heads", heads, kvh, flush=True)
        n, rows, P, lens = 2, 3, 50, [0, 41]
        cache = q3h.Cache(device, n, kvh, hd, P, fmt)
        q = rng.standard_normal((n, rows, heads, hd)).astype(np.float32)
        k = rng.standard_normal((n, rows, kvh, hd)).astype(np.float32)
        v = rng.standard_normal((n, rows, kvh, hd)).astype(np.float32)
        tq = place(q, heads * hd + 3) if heads else None
        got = cache.append(place(k, kvh * hd + 1), place(v, kvh * hd + 5), dev_i(lens), q=tq,
                           q_out=tq, rope=table, q_norm=dev_f(qn) if heads else None,
                           k_norm=dev_f(kn))
        back = [torch.empty((n, rows, kvh, hd), device="cuda") for _ in range(2)]
        cache.read(*back, starts=dev_i(lens))
        for s in range(n):
            for i in range(rows):
                k0 = ref.turned(ref.normed(k[s, i].astype(np.float64), kn, eps), lens[s] + i, hd,
                                False, freq, mag)
                np.testing.assert_array_equal(host(back[0][s, i]),
                                              ref.stored(k0.astype(np.float32), fmt))
                np.testing.assert_array_equal(host(back[1][s, i]), ref.stored(v[s, i], fmt))
                if heads:
                    q0 = ref.turned(ref.normed(q[s, i].astype(np.float64), qn, eps), lens[s] + i,
                                    hd, False, freq, mag)
                    tol = U * np.abs(q0) + 1e-13 * np.abs(q0).max()
                    assert (np.abs(host(got[s, i]).reshape(heads, hd) - q0) <= tol).all()


@pytest.mark.parametrize("fmt", [F, Q])
def test_attend_of_many_sequences(device, fmt):
    """More sequences than lanes: long ones, empty ones, ones without rows, one
    whose length is beyond the bound, one that is none."""
    rng = np.random.default_rng(34)
    n, rows, heads, kvh, hd, P = 150, 3, 4, 2, 64, 900
    lens = rng.integers(0, 300, n)
    lens[[7, 70, 149]] = 890, 850, 870
    lens[[0, 64]] = 0
    counts = rng.integers(0, rows + 1, n)
    counts[[0, 7, 70, 149, 30, 31]] = rows
    parents = random_tree(rng, n, rows)
    k, v = [(rng.standard_normal((n, P, kvh, hd))).astype(np.float32) for _ in range(2)]
    q = rng.standard_normal((n, rows, heads, hd)).astype(np.float32)
    cache = q3h.Cache(device, n, kvh, hd, P, fmt)
    fill(cache, k, v, [P] * n)
    asked = lens.copy()
    asked[30], asked[31] = 896, -1
    out = torch.full((n, rows, heads, hd), 7.0, device="cuda")
    cache.attend(dev_f(q), dev_i(asked), 895, out=out, counts=dev_i(counts),
                 parents=dev_i(parents))
    out = host(out)
    for b in (30, 31):
        assert np.isnan(out[b]).all()
    good = [b for b in range(n) if b not in (30, 31)]
    held = ref.stored(k, fmt).astype(np.float64), ref.stored(v, fmt).astype(np.float64)
    want, bound = ref.attention(q.astype(np.float64), *held, lens, counts, parents, hd ** -0.5)
    for b in good:
        assert (out[b, counts[b]:] == 7).all()
        off = np.abs(out - want)[b, :counts[b]]
        if not (off <= bound[b, :counts[b]]).all():
            at = np.argwhere(off > bound[b, :counts[b]])
            print("sequence", b, lens[b], counts[b], parents[b], len(at), at[:8].tolist(),
                  [(out[b][tuple(i)], want[b][tuple(i)], bound[b][tuple(i)]) for i in at[:8]])
        assert (off <= bound[b, :counts[b]]).all()


def test_graphs_that_share_a_workspace(device):
    """Two captured calls of different shapes over one workspace, replayed in
    turn with eager calls between."""
    rng = np.random.default_rng(35)
    n, kvh, hd, P = 3, 2, 128, 2100
    cache = q3h.Cache(device, n, kvh, hd, P, H)
    base = rng.standard_normal((n, 2000, kvh, hd)).astype(np.float32)
    fill(cache, base, base, [2000, 1990, 700])
    lens = dev_i([1900, 1700, 600])
    calls = []
    need = max(cache.attend_workspace(n, 1, 8, 2000), cache.attend_workspace(n, 17, 16, 2000))
    space = torch.empty(need, dtype=torch.uint8, device="cuda")
    for rows, heads in ((1, 8), (17, 16)):
        q = dev_f(rng.standard_normal((n, rows, heads, hd)))
        out = torch.zeros_like(q)
        parents = dev_i(random_tree(rng, n, rows))

        def call(q=q, out=out, parents=parents):
            cache.attend(q, lens, 2000, out=out, parents=parents, workspace=space)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        calls.append((g, q, out, call))
    for turn in range(4):
        want = []
        for g, q, out, call in calls:
            q.copy_(dev_f(rng.standard_normal(tuple(q.shape))))
            call()
            want.append(out.clone())
            out.zero_()
        torch.cuda.synchronize()
        for g, q, out, call in calls[::1 if turn % 2 else -1]:
            g.replay()
        torch.cuda.synchronize()
        for (g, q, out, call), w in zip(calls, want):
            assert torch.equal(out, w)
        lens += 20


@pytest.mark.parametrize("fmt", [F, H, Q])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,heads", [(1, 2), (3, 10), (40, 6)])
def test_attend_of_rows_between_boundaries(device, fmt, hd, rows, heads):
    """Queries and outputs that begin at odd floats, rows an odd number apart; what
    lies between the rows stays."""
    rng = np.random.default_rng(38)
    n, kvh, P, lens = 2, 2, 1100, [1000, 77]
    cache = q3h.Cache(device, n, kvh, hd, P, fmt)
    k, v = [rng.standard_normal((n, P, kvh, hd)).astype(np.float32) for _ in range(2)]
    q = rng.standard_normal((n, rows, heads, hd)).astype(np.float32)
    fill(cache, k, v, [P] * n)

    def place(ld):
        buf = torch.full((n * rows * ld + 3,), 9.0, device="cuda")
        return buf, buf.as_strided((n, rows, heads * hd), (rows * ld, ld, 1), 3)

    (_, tq), (buf, out) = place(heads * hd + 5), place(heads * hd + 7)
    tq.copy_(dev_f(q).reshape(n, rows, -1))
    cache.attend(tq, dev_i(lens), 1000, out=out)
    held = ref.stored(k, fmt).astype(np.float64), ref.stored(v, fmt).astype(np.float64)
    want, bound = ref.attention(q.astype(np.float64), *held, lens, [rows] * n, None, hd ** -0.5)
    got = host(out).reshape(want.shape)
    assert (np.abs(got - want) <= bound).all()
    out.fill_(9.0)
    assert (host(buf) == 9).all()


@pytest.mark.parametrize("fmt", [F, Q])
@pytest.mark.parametrize("up", [20, 30, 38])
@pytest.mark.parametrize("heads,length", [(1, 40), (24, 40), (2, 3000)])
def test_large_values_of_little_weight_cost_no_precision(device, fmt, up, heads, length):
    """Positions that a row sees, whose values are larger by 2^up and whose weights
    are smaller by more: the others' sum keeps its precision."""
    rng = np.random.default_rng(39)
    hd, P = 64, length + 1
    q = rng.standard_normal((1, 1, heads, hd)).astype(np.float32)
    q[..., 0] = 8
    k = (0.1 * rng.standard_normal((1, P, 1, hd))).astype(np.float32)
    v = rng.standard_normal((1, P, 1, hd)).astype(np.float32)
    for j in range(5, P, 19):
        k[0, j, 0, 0] = -(up + 12) * np.log(2)  # a score of -8 / 8 of it
        v[0, j] *= 2.0 ** up
    cache = q3h.Cache(device, 1, 1, hd, P, fmt)
    fill(cache, k, v, [P])
    held = ref.stored(k, fmt).astype(np.float64), ref.stored(v, fmt).astype(np.float64)
    want, bound = ref.attention(q.astype(np.float64), *held, [length], [1], None, 1 / 8)
    out = host(cache.attend(dev_f(q), dev_i([length]), length, scale=1 / 8))
    ratio = np.abs(out - want) / bound
    print(ratio.max(), flush=True)
    assert (ratio <= 1).all()
