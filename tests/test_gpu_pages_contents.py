"""What the calls on large tables of pages move: reserve beyond the slots of its one launch,
fork beyond its entries, compact beyond its pages. The contents of every sequence are
followed by hand and read back, copied rows and moved pages among them."""
import numpy as np
import pytest
import torch

import pages_ref as pref
import q3h
from test_gpu_draft import dev_f, dev_i

pytestmark = pytest.mark.gpu

F, H, Q, N = q3h.KV_F32, q3h.KV_F16, q3h.KV_Q8, q3h.KV_Q4

# (sequences, positions of one, positions of a page, pages, elements of a head): many short
# sequences, with too few pages and with more than 8192, more of them in use; few of more
# pages than a wave has lanes
SHAPES = [(600, 100, 32, 700, 64), (4500, 128, 32, 17000, 64), (40, 2500, 32, 2500, 128),
          (70, 700, 64, 9000, 64)]


@pytest.mark.parametrize("fmt", [F, H, Q, N])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_contents_of_large_tables(device, shape, fmt):
    n, P, page, pages, hd = SHAPES[shape]
    print(f"{n} sequences of {P}, {pages} pages of {page}, format {fmt}", flush=True)
    rng = np.random.default_rng(100 * shape + fmt)
    kvh, layers, kinds = 2, 2, 509
    cache = q3h.Cache(device, n, kvh, hd, P, fmt, layers=layers, pages=pages, page_positions=page)
    model = pref.Pages(n, pages, page, P)
    # rows of some kinds, and what the format holds of them: [layer][part][kind][head][element]
    rows = rng.standard_normal((layers, 2, kinds, kvh, hd)).astype(np.float32)
    put, held = dev_f(rows), dev_f(pref.stored(rows, fmt))
    # the kind of every position of a sequence, -1: not known; and the sequences' lengths
    known = torch.full((n, P), -1, dtype=torch.int64, device="cuda")
    length = np.zeros(n, int)
    at = torch.arange(P, device="cuda")[None, :]
    copied = moved = shared = 0

    def check():
        for got, want in zip(cache.page_state(),
                             (model.table(), [len(x) for x in model.lists], model.refs())):
            np.testing.assert_array_equal(got.cpu().numpy(), want)
        there = dev_i([min(P, len(x) * page) for x in model.lists])
        for layer in range(layers):
            k = torch.zeros((n, P, kvh, hd), device="cuda")
            v = torch.zeros_like(k)
            cache.read(k, v, counts=there, layer=layer)
            for part, got in enumerate((k, v)):
                same = (got == held[layer, part][known.clamp(min=0)]).flatten(2).all(-1)
                assert bool((same | (known < 0)).all()), (layer, part)
        assert bool(((known >= 0) == (at < dev_i(length)[:, None])).all())

    for turn in range(5):
        # rows to most sequences, behind what they hold
        counts = rng.integers(0, P - length + 1) // rng.choice([1, 1, 4], n)
        counts[rng.random(n) < 0.1] = 0
        most = max(1, int(counts.max()))
        ok = torch.zeros(n, dtype=torch.int32, device="cuda")
        cache.reserve(dev_i(length), most, counts=dev_i(counts), ok=ok)
        want, copies = model.reserve(length.tolist(), counts.tolist())
        np.testing.assert_array_equal(ok.cpu().numpy(), want)
        # (slots that the call can touch, a power of two a sequence: of more than 64 a sequence
        # or 1024 in all not by its one launch)
        slots = 1 << ((most - 1) // page + 1).bit_length()
        if slots > 64 or n * slots > 1024:
            copied += len(copies)
        check()  # (nothing is written yet: copied rows are those that were there)
        counts *= np.array(want)
        kinds_in = torch.from_numpy(rng.integers(0, kinds, (n, most))).cuda()
        for layer in range(layers):
            cache.append(put[layer, 0][kinds_in], put[layer, 1][kinds_in], dev_i(length),
                         counts=dev_i(counts), layer=layer)
        slot = at - dev_i(length)[:, None]
        new = (slot >= 0) & (slot < dev_i(counts)[:, None])
        known = torch.where(new, kinds_in.gather(1, slot.clamp(0, most - 1)), known)
        length += counts
        check()
        # some go on from others, some from an earlier position, some leave
        sources = np.where(rng.random(n) < 0.6, np.arange(n), rng.integers(-1, n, n))
        cut = np.where(sources < 0, 0, length[np.maximum(sources, 0)])
        back = rng.random(n) < 0.3
        cut = np.where(back, (cut * rng.random(n)).astype(int), cut)
        cache.fork(dev_i(sources), dev_i(cut))
        model.fork(sources.tolist(), cut.tolist())
        shared += sum(r > 1 for r in model.refs())
        known = torch.where(at < dev_i(cut)[:, None],
                            known[torch.from_numpy(np.maximum(sources, 0)).cuda()], -1)
        length = cut.copy()
        check()
        gone = rng.random(n) < 0.3
        length[gone] = (length[gone] * rng.random(gone.sum())).astype(int)
        known = torch.where(at < dev_i(length)[:, None], known, -1)
        cache.release(dev_i(length))
        model.release(length.tolist())
        check()
        used, to = model.compact()
        moved += len(to)
        assert cache.compact().item() == used
        check()
    print(f"{copied} pages copied, {moved} moved, {shared} shared", flush=True)
    assert copied > 0 and moved > 0 and shared > 0
