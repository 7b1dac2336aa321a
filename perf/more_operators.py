"""The cases of the operators around the memory of a server's K/V caches: rows
held in 4 bits, caches in pages that sequences share, and rotary positions of
several axes.

Four kinds of case:

- "append": rows' queries and keys normed and rotated by positions of several
  axes (time, height, width), keys and values written to a cache, and the rows
  just written read back as the values that they stand for.
- "attend": rows' attention over a cache in 4 bits, or in pages, each row over
  the positions before the draft and over its own ancestors among the drafted
  rows (a chain: over the rows before it).
- "beams": every prompt's sequence forked into several, a row more reserved for
  each (what they share and are to write is copied), the last pages read back,
  and the forks released.
- "turnover": half of the sequences leave, the pages in use move together, the
  half comes back from a cache that kept it; then the other half. What the
  cache holds in the end is read back.

Formats: "f32", "f16", "q8": one byte per element and one f32 scale per position
and head, scale = max |x| / 127 rounded to f32, byte = x / scale rounded to
even; "q4": D = max |x| / 1785 rounded to f32 per position and head, for each 32
elements a byte s = max |x| / (7 D) rounded up (255 at most), and
n = x / (s D) rounded to even, within -7 .. 7: the value is n s D.

Pages: of page_positions positions each, taken from the lowest free one up, for
the sequences in their order. A page that several sequences hold is replaced by
an own one when a sequence is to write to it; if all that hold it are to, the
first of them keeps it. Pages in use move together: those behind the number of
pages in use, in their order, to the free ones below it, in theirs.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # one token of one sentence, its cache in 4 bits: all latency
        dict(name="append_token_q4", op="append", n=1, rows=1, len=300, heads=16, kv_heads=8,
             head_dim=128, fmt="q4", page=0, rot_dim=128, interleaved=False, axes="dealt"),
        # prompts with pictures into the pages of a server's cache
        dict(name="append_pictures_q4", op="append", n=6, rows=1021, len=4000, heads=32,
             kv_heads=8, head_dim=128, fmt="q4", page=64, rot_dim=128, interleaved=False,
             axes="dealt"),
        # a few rows of many sequences, half of each head turned in pairs of neighbours
        dict(name="append_rows_f16", op="append", n=40, rows=7, len=3001, heads=16, kv_heads=8,
             head_dim=64, fmt="f16", page=32, rot_dim=32, interleaved=True, axes="parts"),
        # one token of one sentence over a cache in 4 bits
        dict(name="attend_token_q4", op="attend", n=1, rows=1, len=171, heads=16, kv_heads=8,
             head_dim=128, fmt="q4", page=0, tree=False),
        # one token of each of a server's 32 sentences
        dict(name="attend_tokens_q4", op="attend", n=32, rows=1, len=4096, heads=16, kv_heads=8,
             head_dim=128, fmt="q4", page=64, tree=False),
        # drafted trees of 12 long sequences, four query heads to a key head
        dict(name="attend_trees_q4", op="attend", n=12, rows=64, len=8000, heads=32, kv_heads=8,
             head_dim=128, fmt="q4", page=0, tree=True),
        # one drafted tree over a long context in pages
        dict(name="attend_tree_pages_f16", op="attend", n=1, rows=27, len=12289, heads=16,
             kv_heads=8, head_dim=128, fmt="f16", page=128, tree=True),
        # prompts behind a shared beginning, in pages of one byte an element
        dict(name="attend_prompts_pages_q8", op="attend", n=2, rows=1500, len=500, heads=16,
             kv_heads=8, head_dim=128, fmt="q8", page=32, tree=False),
        # a short sentence's beams
        dict(name="beams_short_f16", op="beams", n=1, width=4, len=37, layers=5, kv_heads=8,
             head_dim=128, fmt="f16", page=32),
        # 16 prompts, 8 continuations of each
        dict(name="beams_q4", op="beams", n=16, width=8, len=1930, layers=5, kv_heads=8,
             head_dim=128, fmt="q4", page=64),
        # a few short sequences replaced
        dict(name="turnover_f32", op="turnover", n=4, len=61, layers=2, kv_heads=8, head_dim=64,
             fmt="f32", page=32),
        # a server's long sequences replaced
        dict(name="turnover_q8", op="turnover", n=16, len=2051, layers=2, kv_heads=8,
             head_dim=128, fmt="q8", page=64),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "append", "attend", "attend", "attend", "beams", "turnover"))
    heads, kv_heads = rng.choice(((16, 8), (16, 8), (8, 8), (32, 8), (6, 2), (28, 4), (8, 1)))
    hd = rng.choice((128, 128, 64))
    fmt = rng.choice(("f32", "f16", "q8", "q4", "q4", "q4"))
    page = rng.choice((32, 64, 128, 256))
    if op == "beams":
        layers, width = rng.choice((1, 2, 5)), rng.randint(2, 8)
        return dict(op=op, n=_spread(rng, 1, max(1, min(16, 40000 // (layers * width * page)))),
                    width=width, len=_spread(rng, 1, 2000), layers=layers, kv_heads=kv_heads,
                    head_dim=hd, fmt=fmt, page=page)
    if op == "turnover":
        n, layers = _spread(rng, 2, 24), rng.choice((1, 2, 5))
        return dict(op=op, n=n, len=_spread(rng, 1, 60000 // (n * layers)), layers=layers,
                    kv_heads=kv_heads, head_dim=hd, fmt=fmt, page=page)
    if op == "append":
        n = _spread(rng, 1, 40)
        return dict(op=op, n=n, rows=_spread(rng, 1, max(2, 4000 // n)),
                    len=0 if rng.random() < 0.1 else _spread(rng, 1, 8000), heads=heads,
                    kv_heads=kv_heads, head_dim=hd, fmt=fmt, page=rng.choice((0, page)),
                    rot_dim=rng.choice((hd, hd, hd // 2, hd // 4, 20)),
                    interleaved=rng.random() < 0.4, axes=rng.choice(("dealt", "parts")))
    # over contiguous caches of the other formats nothing is new
    page = rng.choice((0, page)) if fmt == "q4" else page
    tree = rng.random() < 0.5
    rows = rng.choice((1, 1, _spread(rng, 2, 64), 0 if tree else _spread(rng, 2, 300)))
    rows = rows or _spread(rng, 2, 64)
    n = _spread(rng, 1, 24)
    most = min(16000, 40000 // n, int(3e6) // (n * rows))
    length = 0 if rng.random() < 0.1 else _spread(rng, 1, max(2, most))
    return dict(op=op, n=n, rows=rows, len=length, heads=heads, kv_heads=kv_heads, head_dim=hd,
                fmt=fmt, page=page, tree=tree and rows <= 64)


def _down(top, n):
    """Lengths of n sequences, longest first: down to a quarter of the longest."""
    return [top - (3 * top * i) // (4 * max(1, n - 1)) if n > 1 else top for i in range(n)]


def _counts(case):
    """Drafted rows of the sequences: from all of them down to a few."""
    n, rows = case["n"], case["rows"]
    return [max(1, rows - rows * i // n) for i in range(n)]


def _pair_axes(case):
    """The axis of each rotated pair: a part of the pairs each (a half, a quarter and what
    is left), or dealt one by one, what is left over to the first axis."""
    pairs = case["rot_dim"] // 2
    each = (5 * pairs) // 16
    if case["axes"] == "parts":
        return [0 if i < pairs - 2 * each else 1 if i < pairs - each else 2 for i in range(pairs)]
    return [i % 3 if i < 3 * each else 0 for i in range(pairs)]


def _positions_of(case):
    """Positions that the cache of a case has for each sequence."""
    return case["len"] + (case["rows"] if case["op"] in ("append", "attend") else 1)


def _pages_of(positions, page):
    return -(-positions // page)


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


def _held(case, seed, n, rows):
    """Keys, with the outlying channels that trained ones have, and values
    [layer][sequence][position][head][element]."""
    kvh, hd, layers = case["kv_heads"], case["head_dim"], case.get("layers", 1)
    wide = torch.exp(0.5 * _normal(_gen(seed, 2), kvh, hd))
    return (_normal(_gen(seed, 3), layers, n, rows, kvh, hd) * wide,
            _normal(_gen(seed, 4), layers, n, rows, kvh, hd))


def _places(host, case):
    """Positions on three axes: text, where all three go on together, and from a
    row of the sequence's own on pictures of up to 30 x 40 patches, where the time stands."""
    n, rows = case["n"], case["rows"]
    top = max(1, _positions_of(case) - 1)
    out = np.zeros((3, n, rows), np.int64)
    for b, start in enumerate(host.randint(0, case["len"] + 1, n)):
        t = np.arange(rows)
        at = host.randint(0, rows)
        tall, wide = host.randint(1, 31), host.randint(1, 41)
        patch = np.maximum(t - at, 0)
        shot = patch // (tall * wide)
        text = np.minimum(t, at)
        out[0, b] = start + text + shot
        out[1, b] = start + text + np.where(t < at, 0, patch // wide % tall)
        out[2, b] = start + text + np.where(t < at, 0, patch % wide)
    return np.minimum(out, top).astype(np.int32)


def _inputs(case, seed):
    """The case's inputs: what both forms and exact() start from."""
    host = np.random.RandomState(int(seed) % (1 << 31))
    op, n = case["op"], case["n"]
    x = {}
    lens = np.array(_down(case["len"], n))[host.permutation(n)]
    x["lens"] = _ints(lens)
    if op == "beams":
        w = case["width"]
        x["k"], x["v"] = _held(case, seed, n, case["len"])
        # sequence b continues prompt b % n
        x["sources"] = _ints(np.arange(n * w) % n)
        x["forked"] = _ints(np.tile(lens, w))
        x["left"] = _ints(np.concatenate([lens, np.zeros(n * (w - 1), np.int64)]))
        x["starts"] = _ints(np.tile(lens // case["page"] * case["page"], w))
        x["tails"] = _ints(np.tile(lens % case["page"], w))
        return x
    if op == "turnover":
        x["k"], x["v"] = _held(case, seed, n, case["len"])
        odd = np.arange(n) % 2
        half = host.permutation(odd)
        x["sources"] = [_ints(np.where(half == g, np.arange(n), -1)) for g in (0, 1)]
        x["stay"] = [_ints(np.where(half == g, 0, lens)) for g in (0, 1)]
        x["come"] = [_ints(np.where(half == g, lens, 0)) for g in (0, 1)]
        x["zero"] = _ints(np.zeros(n, np.int64))
        return x
    rows, h, kvh, hd = case["rows"], case["heads"], case["kv_heads"], case["head_dim"]
    x["counts"] = _ints(np.array(_counts(case))[host.permutation(n)])
    if op == "append":
        x["qkv"] = _normal(_gen(seed, 5), n, rows, (h + 2 * kvh) * hd)
        x["q_norm"] = 1 + 0.1 * _normal(_gen(seed, 6), hd)
        x["k_norm"] = torch.exp(0.5 * _normal(_gen(seed, 7), hd))
        x["places"] = _ints(_places(host, case))
        return x
    # a node's parent: most often one of the last few, at times none of them
    back = host.geometric(0.4, (n, rows))
    parents = np.maximum(np.arange(rows)[None, :] - back, -1) if case["tree"] else \
        np.broadcast_to(np.arange(rows)[None, :] - 1, (n, rows))
    x["parents"] = _ints(np.ascontiguousarray(parents))
    x["q"] = _normal(_gen(seed, 5), n, rows, h, hd)
    k, v = _held(case, seed, n, case["len"] + rows)
    x["k"], x["v"] = k[0], v[0]
    return x


# ---------------------------------------------------------------------------
# the framework's caches and operators


def _package():
    path = os.path.join(ROOT, "mormot2-qwen-tts_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import q3h
    return q3h


def _own_cache(case, dev, sequences, positions, page, spare=0):
    q3h = _package()
    fmt = {"f32": q3h.KV_F32, "f16": q3h.KV_F16, "q8": q3h.KV_Q8, "q4": q3h.KV_Q4}[case["fmt"]]
    paged = {}
    if page:
        paged = dict(page_positions=page, pages=sequences * _pages_of(positions, page) + spare)
    return q3h.Cache(dev, sequences, case["kv_heads"], case["head_dim"], positions, fmt,
                     layers=case.get("layers", 1), **paged)


def _own_fill(case, cache, k, v, held):
    """Rows [layer][sequence] from position 0 on; pages in the order that sequences
    growing together take them."""
    zero = torch.zeros_like(held)
    page = case["page"]
    if page:
        rows = k.shape[2]
        for at in range(page, rows + page, page):
            cache.reserve(zero, rows, counts=held.clamp(max=at))
    for layer in range(k.shape[0]):
        cache.append(k[layer], v[layer], zero, counts=held, layer=layer)


def _prepare_own(case, x, state):
    q3h = _package()
    dev = state["dev"] = q3h.Device(0)
    op, n, page = case["op"], case["n"], case["page"]
    if op == "beams":
        # (a page's positions at least: so many rows are read of each sequence)
        cache = state["cache"] = _own_cache(case, dev, n * case["width"],
                                            max(case["len"] + 1, page), page)
        _own_fill(case, cache, x["k"], x["v"], x["lens"])
        state["ok"] = torch.zeros(n * case["width"], dtype=torch.int32, device="cuda")
        return
    if op == "turnover":
        cache = state["cache"] = _own_cache(case, dev, n, case["len"], page)
        store = state["store"] = _own_cache(case, dev, n, case["len"], 0)
        for layer in range(case["layers"]):
            store.append(x["k"][layer], x["v"][layer], x["zero"], counts=x["lens"], layer=layer)
        _turnover_own(state, x)
        return
    positions = _positions_of(case)
    cache = state["cache"] = _own_cache(case, dev, n, positions, page)
    held = x["lens"] + x["counts"]
    if op == "attend":
        _own_fill(case, cache, x["k"][None], x["v"][None], held)
        return
    state["rope"] = q3h.Rope(dev, case["head_dim"], positions, THETA, rot_dim=case["rot_dim"],
                             interleaved=case["interleaved"], axes=_pair_axes(case))
    if page:
        cache.reserve(torch.zeros_like(held), positions, counts=held)


def _turnover_own(state, x):
    cache, used = state["cache"], []
    for g in (0, 1):
        cache.release(x["stay"][g])
        used.append(cache.compact())
        cache.reserve(x["zero"], state["case"]["len"], counts=x["come"][g])
        cache.copy(state["store"], x["sources"][g], x["lens"])
    return used


def _run_own(state):
    case, x, cache = state["case"], state["x"], state["cache"]
    op = case["op"]
    if op == "attend":
        parents = x["parents"] if case["tree"] else None
        cache.attend(x["q"], x["lens"], case["len"], out=state["q_out"], counts=x["counts"],
                     parents=parents)
        return {"out": state["q_out"]}
    k, v = state["k_out"], state["v_out"]
    if op == "append":
        h, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
        xq, xk, xv = x["qkv"].split((h * hd, kvh * hd, kvh * hd), dim=-1)
        cache.append(xk, xv, x["lens"], counts=x["counts"], q=xq, q_out=state["q_out"],
                     rope=state["rope"], positions=x["places"], q_norm=x["q_norm"],
                     k_norm=x["k_norm"], eps=EPS)
        cache.read(k, v, starts=x["lens"], counts=x["counts"])
        return {"q": state["q_out"], "k": k, "v": v}
    if op == "beams":
        cache.fork(x["sources"], x["forked"])
        cache.reserve(x["forked"], 1, ok=state["ok"])
        for layer in range(case["layers"]):
            cache.read(k[layer], v[layer], starts=x["starts"], counts=x["tails"], layer=layer)
        table, counts, refs = cache.page_state()
        cache.release(x["left"])
        return {"k": k, "v": v, "ok": state["ok"], "table": table, "counts": counts, "refs": refs}
    used = _turnover_own(state, x)
    for layer in range(case["layers"]):
        cache.read(k[layer], v[layer], counts=x["lens"], layer=layer)
    table, counts, refs = cache.page_state()
    return {"k": k, "v": v, "used": used, "table": table, "counts": counts, "refs": refs}


# ---------------------------------------------------------------------------
# the plain forms: what a format holds of rows, caches as tensors
# [page][layer][head][position][element] and one page more, where goes what is not
# kept (a cache without pages has one of all positions for each sequence)


def _stored(rows, fmt):
    """f32 rows as the format holds them: (elements, scales)."""
    if fmt == "f32":
        return rows, None
    if fmt == "f16":
        return rows.to(torch.float16), None
    wide = rows.double()
    most = wide.abs().amax(-1, keepdim=True)
    if fmt == "q8":
        scale = (most / 127).float()
        return torch.round(wide / scale.double()).to(torch.int8), scale
    d = (most / 1785).float()
    groups = wide.unflatten(-1, (-1, 32))
    s = torch.ceil(groups.abs().amax(-1) / (7 * d.double())).clamp(max=255)
    step = (s * d.double())[..., None]
    n = torch.where(step > 0, torch.round(groups / step), 0).clamp(-7, 7)
    return (n * s[..., None]).flatten(-2).to(torch.int16), d


class _Plain:
    """A cache in its plain form."""

    def __init__(self, case, sequences, positions, page):
        self.fmt, self.page = case["fmt"], page or positions
        self.most = _pages_of(positions, self.page)
        self.pages = sequences * self.most
        kind = {"f32": torch.float32, "f16": torch.float16, "q8": torch.int8,
                "q4": torch.int16}[self.fmt]
        shape = (self.pages + 1, case.get("layers", 1), case["kv_heads"], self.page)
        hd = case["head_dim"]
        self.parts = {"k": torch.zeros(*shape, hd, dtype=kind, device="cuda"),
                      "v": torch.zeros(*shape, hd, dtype=kind, device="cuda")}
        if self.fmt in ("q8", "q4"):
            self.parts["ks"] = torch.zeros(*shape, 1, device="cuda")
            self.parts["vs"] = torch.zeros(*shape, 1, device="cuda")
        self.table = torch.full((sequences, self.most), -1, dtype=torch.int64, device="cuda")
        self.counts = torch.zeros(sequences, dtype=torch.int64, device="cuda")
        self.refs = torch.zeros(self.pages + 1, dtype=torch.int64, device="cuda")
        if not page:
            self.table[:, 0] = torch.arange(sequences, device="cuda")

    def where(self, at):
        """Positions [sequence][row] as (page, position in it); below 0: the page more."""
        slot = (at // self.page).clamp(0, self.most - 1)
        page = torch.gather(self.table[:at.shape[0]], 1, slot)
        return torch.where((at >= 0) & (page >= 0), page, self.pages), at % self.page

    def put(self, at, k, v, layer=0):
        page, off = self.where(at)
        for part, rows in (("k", k), ("v", v)):
            elements, scales = _stored(rows, self.fmt)
            self.parts[part][page, layer, :, off] = elements
            if scales is not None:
                self.parts[part + "s"][page, layer, :, off] = scales

    def rows(self, part, at, layer=0):
        """f32 rows [sequence][row][head][element] at positions [sequence][row]."""
        page, off = self.where(at)
        rows = self.parts[part][page, layer, :, off].float()
        if part + "s" in self.parts:
            rows = rows * self.parts[part + "s"][page, layer, :, off]
        return rows

    def all(self, part, positions):
        """f32 rows [sequence][head][position][element] of the first positions."""
        page = torch.where(self.table >= 0, self.table, self.pages)
        rows = self.parts[part][page, 0].float()
        if part + "s" in self.parts:
            rows = rows * self.parts[part + "s"][page, 0]
        return rows.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :positions]

    def _hold(self, pages, more):
        """more added to the holders of pages (negative ones: none)."""
        pages = torch.where(pages >= 0, pages, self.pages).flatten()
        self.refs.scatter_add_(0, pages, torch.full_like(pages, more))
        self.refs[self.pages] = 0

    def fork(self, sources, lens):
        n = sources.shape[0]
        slot = torch.arange(self.most, device="cuda")
        counts = -(-lens.long() // self.page)
        new = torch.where(slot < counts[:, None], self.table[sources.long()], -1)
        self._hold(new, 1)
        self._hold(self.table[:n], -1)
        self.table[:n] = new
        self.counts[:n] = counts

    def release(self, lens):
        n = lens.shape[0]
        slot = torch.arange(self.most, device="cuda")
        counts = torch.minimum(self.counts[:n], -(-lens.long() // self.page))
        gone = slot >= counts[:, None]
        self._hold(torch.where(gone, self.table[:n], -1), -1)
        self.table[:n] = torch.where(gone, -1, self.table[:n])
        self.counts[:n] = counts

    def reserve(self, lens, counts):
        """Pages for positions lens .. lens + counts - 1 of the first sequences."""
        n = lens.shape[0]
        lens, counts = lens.long()[:, None], counts.long()[:, None]
        table, held = self.table[:n], self.counts[:n, None]
        slot = torch.arange(self.most, device="cuda")
        first, end = lens // self.page, -(-(lens + counts) // self.page)
        end = torch.where(counts > 0, end, 0)
        at = torch.where(table >= 0, table, self.pages)
        shared = (slot >= first) & (slot < torch.minimum(held, end)) & (self.refs[at] > 1)
        # who keeps a page that all its holders are to write to
        number = torch.arange(n, device="cuda")[:, None].expand_as(at)
        page = torch.where(shared, at, self.pages).flatten()
        writers = torch.zeros_like(self.refs).scatter_add_(0, page, torch.ones_like(page))
        lowest = torch.full_like(self.refs, n).scatter_reduce_(0, page, number.flatten(), "amin")
        keeps = shared & (writers == self.refs)[at] & (lowest[at] == number)
        take = (shared & ~keeps) | ((slot >= held) & (slot < end))
        wanted = take.sum(1)
        upto = wanted.cumsum(0)
        free = self.refs[:self.pages] == 0
        order = torch.sort(free.int(), descending=True, stable=True).indices
        ok = (wanted == 0) | (upto <= free.sum())
        rank = (upto - wanted)[:, None] + take.cumsum(1) - 1
        take = take & ok[:, None]
        new = torch.where(take, order[rank.clamp(0, self.pages - 1)], -1)
        self._hold(new, 1)
        self._hold(torch.where(take & shared, table, -1), -1)
        # the positions before lens of a page that is replaced
        copied = take & shared & (slot == first) & (lens % self.page > 0)
        src = torch.where(copied, at, self.pages).amin(1)
        dst = torch.where(copied, new, self.pages).amin(1)
        for part in self.parts.values():
            part[dst] = part[src]
        self.table[:n] = torch.where(take, new, table)
        self.counts[:n] = torch.where(ok, torch.maximum(self.counts[:n], end[:, 0]),
                                      self.counts[:n])
        still = (slot >= first) & (slot < end) & (self.refs[self.table[:n]] > 1)
        return (ok & ~still.any(1)).int()

    def compact(self):
        used = self.refs[:self.pages] > 0
        number = torch.arange(self.pages, device="cuda")
        n = used.sum()
        hole, mover = ~used & (number < n), used & (number >= n)
        # the k-th mover to the k-th hole
        holes = torch.sort(hole.int(), descending=True, stable=True).indices
        movers = torch.sort(mover.int(), descending=True, stable=True).indices
        to = torch.where(mover, holes[(mover.cumsum(0) - 1).clamp(min=0)], number)
        source = torch.where(hole, movers[(hole.cumsum(0) - 1).clamp(min=0)], number)
        for part in self.parts.values():
            part[:self.pages] = part[source]
        self.refs[:self.pages] = torch.where(number < n, self.refs[source], 0)
        self.table = torch.where(self.table >= 0, to[self.table.clamp(min=0)], -1)
        return n.int()[None]

    def copy(self, src, sources, lens, positions):
        at = torch.arange(positions, device="cuda")[None, :].expand(sources.shape[0], -1)
        at = torch.where((at < lens[:, None]) & (sources[:, None] >= 0), at, -1)
        page, off = self.where(at)
        from_page, from_off = src.where(at)
        for part in self.parts:
            self.parts[part][page, :, :, off] = src.parts[part][from_page, :, :, from_off]

    def state(self):
        return {"table": self.table.int(), "counts": self.counts.int(),
                "refs": self.refs[:self.pages].int()}


def _span(n, rows, starts, counts):
    """Positions [sequence][row], -1 behind a sequence's rows."""
    t = torch.arange(rows, device="cuda")[None, :].expand(n, -1)
    return torch.where(t < counts[:, None], starts[:, None] + t, -1)


def _prepare_plain(case, x, state):
    op, n, page = case["op"], case["n"], case["page"]
    if op == "beams":
        cache = state["cache"] = _Plain(case, n * case["width"], case["len"] + 1, page)
    elif op == "turnover":
        cache = state["cache"] = _Plain(case, n, case["len"], page)
        state["store"] = _Plain(case, n, case["len"], 0)
        for layer in range(case["layers"]):
            state["store"].put(_span(n, case["len"], x["zero"], x["lens"]), x["k"][layer],
                               x["v"][layer], layer)
        _turnover_plain(state, x)
        return
    else:
        cache = state["cache"] = _Plain(case, n, _positions_of(case), page)
    held = x["lens"] if op == "beams" else x["lens"] + x["counts"]
    zero = torch.zeros_like(held)
    if page:
        most = case["len"] + (0 if op == "beams" else case["rows"])
        for at in [most] if op == "append" else range(page, most + page, page):
            cache.reserve(zero, held.clamp(max=at))
    if op == "append":
        return
    ks, vs = (x["k"], x["v"]) if op == "beams" else (x["k"][None], x["v"][None])
    for layer in range(ks.shape[0]):
        at = _span(n, ks.shape[2], zero, held)
        if cache.table.shape[0] > n:  # (the forks hold nothing yet)
            more = cache.table.shape[0] - n
            at = torch.cat((at, torch.full((more, at.shape[1]), -1, device="cuda")))
            pad = torch.zeros(more, *ks.shape[2:], device="cuda")
            cache.put(at, torch.cat((ks[layer], pad)), torch.cat((vs[layer], pad)), layer)
        else:
            cache.put(at, ks[layer], vs[layer], layer)


def _turnover_plain(state, x):
    cache, used = state["cache"], []
    for g in (0, 1):
        cache.release(x["stay"][g])
        used.append(cache.compact())
        cache.reserve(x["zero"], x["come"][g])
        cache.copy(state["store"], x["sources"][g], x["lens"], state["case"]["len"])
    return used


def _normed(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()


def _rotated(x, case, angle):
    cos, sin = angle.cos()[:, :, None, :], angle.sin()[:, :, None, :]
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
    pairs = torch.arange(case["rot_dim"] // 2, dtype=torch.float64, device="cuda")
    angle = x["places"].double()[state["axes"]].permute(1, 2, 0) * \
        THETA ** (-2.0 * pairs / case["rot_dim"])
    at = _span(n, rows, x["lens"], x["counts"])
    qkv = x["qkv"].view(n, rows, h + 2 * kvh, hd)
    q, k, v = qkv[:, :, :h].double(), qkv[:, :, h:h + kvh].double(), qkv[:, :, h + kvh:]
    q = _rotated(_normed(q, x["q_norm"]), case, angle)
    k = _rotated(_normed(k, x["k_norm"]), case, angle)
    cache.put(at, k, v)
    keep = (at >= 0)[:, :, None, None]
    return {"q": torch.where(keep, q, 0), "k": torch.where(keep, cache.rows("k", at), 0),
            "v": torch.where(keep, cache.rows("v", at), 0)}


def _square(reach):
    return (reach @ reach).clamp(max=1)


def _ancestors(parents):
    """[sequence][row][row]: whether a row is the other one or comes after it on its path
    (of at most 64 rows: each squaring doubles the steps that are followed)."""
    rows = parents.shape[1]
    t = torch.arange(rows, device="cuda", dtype=torch.int32)
    step = ((parents[:, :, None] == t) | (t[:, None] == t)).float()
    return _square(_square(_square(_square(_square(_square(step)))))) > 0


def _run_attend(state):
    case, x, cache = state["case"], state["x"], state["cache"]
    n, rows, h, kvh, hd = (case[k] for k in ("n", "rows", "heads", "kv_heads", "head_dim"))
    positions, g = case["len"] + rows, h // kvh
    lens, counts = x["lens"][:, None, None], x["counts"][:, None, None]
    k, v = cache.all("k", positions), cache.all("v", positions)
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


def _read_back(case, cache, at):
    keep = (at >= 0)[:, :, None, None]
    return {part: torch.stack([torch.where(keep, cache.rows(part, at, layer), 0)
                               for layer in range(case["layers"])]) for part in ("k", "v")}


def _run_beams(state):
    case, x, cache = state["case"], state["x"], state["cache"]
    cache.fork(x["sources"], x["forked"])
    ok = cache.reserve(x["forked"], torch.ones_like(x["forked"]))
    at = _span(case["n"] * case["width"], case["page"], x["starts"], x["tails"])
    answer = _read_back(case, cache, at)
    answer.update(cache.state(), ok=ok)
    cache.release(x["left"])
    return answer


def _run_turnover(state):
    case, x, cache = state["case"], state["x"], state["cache"]
    used = _turnover_plain(state, x)
    answer = _read_back(case, cache, _span(case["n"], case["len"], x["zero"], x["lens"]))
    answer.update(cache.state(), used=used)
    return answer


# ---------------------------------------------------------------------------


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": case, "x": x}
    (_prepare_own if own else _prepare_plain)(case, x, state)
    x.pop("k", None), x.pop("v", None)
    op, n, hd = case["op"], case["n"], case["head_dim"]
    if op == "append":
        state["axes"] = torch.tensor(_pair_axes(case), device="cuda")
    # the buffers of a program's outputs, rows of no sequence zero
    if op in ("append", "attend"):
        state["q_out"] = torch.zeros(n, case["rows"], case["heads"], hd, device="cuda")
    if op != "attend":
        shape = {"append": (n, case.get("rows")), "turnover": (case.get("layers"), n, case["len"]),
                 "beams": (case.get("layers"), n * case.get("width", 0), case["page"])}[op]
        state["k_out"] = torch.zeros(*shape, case["kv_heads"], hd, device="cuda")
        state["v_out"] = torch.zeros(*shape, case["kv_heads"], hd, device="cuda")
    return state


def run(state):
    if own:
        return _run_own(state)
    return {"append": _run_append, "attend": _run_attend, "beams": _run_beams,
            "turnover": _run_turnover}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    op, kvh, hd = case["op"], case["kv_heads"], case["head_dim"]
    # bytes of a position's keys and values in the format, and as f32
    held = 2 * kvh * {"f32": 4 * hd, "f16": 2 * hd, "q8": hd + 4, "q4": hd // 2 + hd // 32 + 4}[
        case["fmt"]]
    wide = 8 * kvh * hd
    lens = _down(case["len"], case["n"])
    if op == "beams":
        page, w, layers = case["page"], case["width"], case["layers"]
        tails = sum(n % page for n in lens)
        table = sum(_pages_of(n + 1, page) for n in lens) * w
        pages = case["n"] * w * _pages_of(case["len"] + 1, page)
        return {"bytes": layers * tails * ((w - 1) * 2 * held + w * (held + wide)) +
                8 * table + 8 * pages, "flops": 2 * layers * tails * w * kvh * hd}
    if op == "turnover":
        page, layers = case["page"], case["layers"]
        pages = sorted(_pages_of(n, page) for n in lens)
        # the smaller half's pages move twice (which sequences it has goes by the seed: the
        # mean), and every position is copied and read once
        moved = 2 * (sum(pages) * (case["n"] // 2) // case["n"]) * page
        return {"bytes": layers * (2 * moved * held + sum(lens) * (3 * held + wide)) +
                16 * sum(pages), "flops": 2 * layers * sum(lens) * kvh * hd}
    h, counts = case["heads"], _counts(case)
    rows = sum(counts)
    if op == "append":
        return {"bytes": rows * (4 * (2 * h + 2 * kvh) * hd + 2 * held + wide + 12),
                "flops": rows * (10 * (h + kvh) + 4 * kvh) * hd}
    # the pairing of lengths and counts goes by the seed: their means
    mean = sum(lens) / case["n"] + (0 if case["tree"] else case["rows"] / 4)
    return {"bytes": int(sum(lens) + rows) * held + 8 * rows * h * hd,
            "flops": int(4 * rows * (mean + 1) * h * hd)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def _exact_values(rows, fmt):
    """What the format holds of f32 rows, in float64 (numpy)."""
    if fmt == "f16":
        return rows.astype(np.float16).astype(np.float64)
    wide = rows.astype(np.float64)
    if fmt == "f32" or wide.size == 0:
        return wide
    most = np.abs(wide).max(-1, keepdims=True)
    if fmt == "q8":
        scale = (most / 127).astype(np.float32).astype(np.float64)
        return np.rint(wide / scale) * scale
    d = (most / 1785).astype(np.float32).astype(np.float64)
    out = np.empty_like(wide)
    for at in range(0, wide.shape[-1], 32):
        part = wide[..., at:at + 32]
        s = np.minimum(255, np.ceil(np.abs(part).max(-1, keepdims=True) / (7 * d)))
        step = np.where(s > 0, s * d, 1)
        out[..., at:at + 32] = np.clip(np.rint(part / step), -7, 7) * (s * d)
    return out


def _exact_append(case, x):
    n, rows, h, kvh, hd = (case[k] for k in ("n", "rows", "heads", "kv_heads", "head_dim"))
    d = case["rot_dim"]
    qkv = x["qkv"].cpu().numpy().reshape(n, rows, h + 2 * kvh, hd)
    weight = np.concatenate([np.repeat(x["q_norm"].cpu().numpy()[None], h, 0),
                             np.repeat(x["k_norm"].cpu().numpy()[None], kvh, 0)]).astype(np.float64)
    counts, places = x["counts"].cpu().numpy(), x["places"].cpu().numpy()
    freq = np.array([math.exp(-2.0 * i / d * math.log(THETA)) for i in range(d // 2)])
    axes = _pair_axes(case)
    out = {"q": np.zeros((n, rows, h, hd)), "k": np.zeros((n, rows, kvh, hd)),
           "v": np.zeros((n, rows, kvh, hd))}
    for b in range(n):
        c = int(counts[b])
        y = qkv[b, :c, :h + kvh].astype(np.float64)
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + EPS) * weight
        turn = np.exp(1j * (places[axes, b, :c].T * freq))[:, None, :]
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
            for t in range(c):
                p = t
                while p >= 0:
                    sees[t, length + p] = True
                    p = int(parents[b, p])
        else:
            sees[:, length:] = np.tri(c, dtype=bool)
        hidden = torch.from_numpy(~sees).cuda()
        k, v = (torch.from_numpy(_exact_values(x[p][b, :length + c].cpu().numpy(),
                                               case["fmt"])).cuda() for p in ("k", "v"))
        for head in range(h):
            z = x["q"][b, :c, head].double().matmul(k[:, head // g].t()) / math.sqrt(hd)
            z = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
            out[b, :c, head] = z.matmul(v[:, head // g].contiguous())
    return {"out": out}


class _Pages:
    """A cache's pages as lists."""

    def __init__(self, sequences, pages, page):
        self.page, self.lists, self.refs = page, [[] for _ in range(sequences)], [0] * pages

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def reserve(self, starts, ends):
        """Enough pages for all: one sequence after another, who comes last to a page that
        its other holders left keeps it; but the first of the call does if all leave."""
        touched = [range(s // self.page, min(len(held), _pages_of(e, self.page))) if e > s else ()
                   for held, s, e in zip(self.lists, starts, ends)]
        writers = {}
        for b, slots in enumerate(touched):
            for i in slots:
                writers.setdefault(self.lists[b][i], []).append(b)
        keeps = {p: who[0] for p, who in writers.items() if len(who) == self.refs[p]}
        shared = {p for p in writers if self.refs[p] > 1}
        left = []
        for b, slots in enumerate(touched):
            for i in slots:
                p = self.lists[b][i]
                if p in shared and keeps.get(p) != b:
                    self.lists[b][i] = self.take()
                    left.append(p)
            if ends[b] > starts[b]:
                while len(self.lists[b]) < _pages_of(ends[b], self.page):
                    self.lists[b].append(self.take())
        for p in left:
            self.refs[p] -= 1

    def cut(self, b, positions):
        while len(self.lists[b]) > _pages_of(positions, self.page):
            self.refs[self.lists[b].pop()] -= 1

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        holes = [p for p in range(used) if not self.refs[p]]
        movers = [p for p in range(used, len(self.refs)) if self.refs[p]]
        to = dict(zip(movers, holes))
        for p, h in to.items():
            self.refs[h], self.refs[p] = self.refs[p], 0
        self.lists = [[to.get(p, p) for p in held] for held in self.lists]
        return used

    def state(self, most):
        return {"table": np.array([held + [-1] * (most - len(held)) for held in self.lists]),
                "counts": np.array([len(held) for held in self.lists]),
                "refs": np.array(self.refs)}


def _exact_beams(case, x):
    n, w, page = case["n"], case["width"], case["page"]
    lens = x["lens"].cpu().tolist()
    most = _pages_of(case["len"] + 1, page)
    pages = _Pages(n * w, n * w * most, page)
    for at in range(page, case["len"] + page, page):
        for b in range(n):
            pages.reserve([0] * (n * w), [min(lens[i], at) if i == b else 0 for i in range(n * w)])
    for b in range(n, n * w):
        pages.lists[b] = list(pages.lists[b % n])
        for p in pages.lists[b]:
            pages.refs[p] += 1
    pages.reserve(lens * w, [a + 1 for a in lens] * w)
    answer = dict(pages.state(most), ok=np.ones(n * w, np.int64))
    for part in ("k", "v"):
        rows = x[part].cpu().numpy()
        out = answer[part] = np.zeros((case["layers"], n * w, page, *rows.shape[3:]))
        for b in range(n * w):
            start = lens[b % n] // page * page
            out[:, b, :lens[b % n] - start] = _exact_values(rows[:, b % n, start:lens[b % n]],
                                                            case["fmt"])
    return answer


def _exact_turnover(case, x):
    n, page = case["n"], case["page"]
    lens = x["lens"].cpu().tolist()
    most = _pages_of(case["len"], page)
    pages = _Pages(n, n * most, page)
    halves = [(s >= 0).cpu().tolist() for s in x["sources"]]
    for _ in range(2):  # (once before the pass)
        used = []
        for half in halves:
            for b in range(n):
                if half[b]:
                    pages.cut(b, 0)
            used.append(np.array([pages.compact()]))
            pages.reserve([0] * n, [lens[b] if half[b] else 0 for b in range(n)])
    answer = dict(pages.state(most), used=used)
    for part in ("k", "v"):
        rows = x[part].cpu().numpy()
        out = answer[part] = np.zeros(rows.shape)
        for b in range(n):
            out[:, b, :lens[b]] = _exact_values(rows[:, b, :lens[b]], case["fmt"])
    return answer


def exact(case, seed):
    x = _inputs(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "beams": _exact_beams,
            "turnover": _exact_turnover}[case["op"]](case, x)
