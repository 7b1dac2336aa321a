"""Caches in pages at the edges of what their calls take: lengths between a cache's last
position and the end of its last page, calls without rows, tables of just the size that is
forked in one launch and of more."""
import gc

import numpy as np
import pytest
import torch

import pages_ref as pref
import q3h
from test_gpu_draft import dev_i

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_handles_left():
    """Handles that a refusal's traceback still holds go before the device does."""
    yield
    gc.collect()


@pytest.mark.parametrize("sequences", [4, 1500])
@pytest.mark.parametrize("positions,page", [(100, 32), (97, 64), (1, 256), (129, 128)])
def test_fork_beyond_the_cache(device, sequences, positions, page):
    """A length that the source's last page reaches and the cache's positions do not leaves
    its sequence as it is: of few sequences in one launch, of many in two."""
    print(f"fork of {sequences} sequences of {positions} in pages of {page}", flush=True)
    slots = -(-positions // page)
    cache = q3h.Cache(device, sequences, 1, 64, positions, q3h.KV_F16, pages=3 * slots,
                      page_positions=page)
    zero = np.zeros(sequences, int)
    counts = zero.copy()
    counts[:2] = positions, 1
    cache.reserve(dev_i(zero), positions, counts=dev_i(counts))
    before = [t.cpu().numpy() for t in cache.page_state()]
    assert before[1][:2].tolist() == [slots, 1]
    most = slots * page
    for length in (positions + 1, most, most + 1, 2 ** 31 - 1):
        sources, lens = np.full(sequences, -2), zero.copy()
        sources[:3], lens[:3] = 0, length
        cache.fork(dev_i(sources), dev_i(lens))
        for was, now in zip(before, cache.page_state()):
            np.testing.assert_array_equal(was, now.cpu().numpy(), err_msg=str(length))
    sources, lens = np.full(sequences, -2), zero.copy()
    sources[1], lens[1] = 0, positions
    cache.fork(dev_i(sources), dev_i(lens))
    table, held, refs = [t.cpu().numpy() for t in cache.page_state()]
    np.testing.assert_array_equal(table[1], table[0])
    assert held[1] == slots and (refs[table[0]] == 2).all()


def test_append_of_no_rows_at_positions(device):
    """A step in which no sequence has a row: tensors without elements, which have no address."""
    rope = q3h.Rope(device, 64, 100, 1e4, axes=[i % 3 for i in range(32)])
    for pages in (0, 4):
        cache = q3h.Cache(device, 2, 2, 64, 100, q3h.KV_Q4, pages=pages, page_positions=32)
        for n, rows in ((2, 0), (0, 3)):
            x = torch.zeros((n, rows, 2, 64), device="cuda")
            at = torch.zeros((3, n, rows), dtype=torch.int32, device="cuda")
            q = cache.append(x, x, dev_i(np.zeros(n)), q=x, rope=rope, positions=at)
            assert q.shape == x.shape
            cache.append(x, x, dev_i(np.zeros(n)), rope=rope)


@pytest.mark.parametrize("n,slots", [(1024, 4), (1023, 5), (1025, 3), (64, 64), (65, 64), (63, 65),
                                     (1, 4096), (1, 4097), (3, 1365), (300, 40)])
def test_forks_of_any_size(device, n, slots):
    """Any assignment of sequences, a few times over, against lists."""
    print(f"fork of {n} sequences of {slots} pages", flush=True)
    rng = np.random.default_rng(n + slots)
    P, pages = 32 * slots, n * slots + 5
    cache = q3h.Cache(device, n, 1, 64, P, q3h.KV_Q4, pages=pages, page_positions=32)
    model = pref.Pages(n, pages, 32, P)
    counts = rng.integers(0, P + 1, n)
    counts[rng.integers(0, n)] = P
    cache.reserve(dev_i(np.zeros(n)), P, counts=dev_i(counts))
    model.reserve([0] * n, counts.tolist())
    for m in (n, n, max(1, n // 2), n):
        sources = rng.integers(-1, n, m)
        sources[rng.random(m) < 0.3] = 0
        own = rng.random(m) < 0.3
        sources[own] = np.arange(m)[own]
        room = np.array([len(model.lists[s]) * 32 if s >= 0 else 0 for s in sources])
        lens = np.where(rng.random(m) < 0.5, room, (room * rng.random(m)).astype(int))
        cache.fork(dev_i(sources), dev_i(lens))
        model.fork(sources.tolist(), lens.tolist())
        for got, want in zip(cache.page_state(),
                             (model.table(), [len(x) for x in model.lists], model.refs())):
            np.testing.assert_array_equal(got.cpu().numpy(), want)
