"""Caches in 4 bits, in pages, and rotary positions of several axes, from their
definitions: numpy and lists."""
import numpy as np

import draft_ref as ref

Q4 = 4


def stored(x, fmt):
    """What a format holds of f32 rows, as float32 (draft_ref.stored, and 4 bits)."""
    if fmt != Q4:
        return ref.stored(x, fmt)
    x = np.asarray(x, np.float32)
    wide = x.astype(np.float64).reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        scale = (np.abs(wide).max((-2, -1), keepdims=True) / 1785).astype(np.float32)
        d = scale.astype(np.float64)
        step = np.minimum(255, np.ceil(np.abs(wide).max(-1, keepdims=True) / (7 * d)))
        n = np.clip(np.rint(wide / (step * d)), -7, 7)
        some = (scale > 0) & (step > 0)
        out = np.where(some, n * step, 0).astype(np.float32) * np.where(some, scale, np.float32(0))
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    return np.where(bad, np.float32(np.nan), out.reshape(x.shape))


def turned(x, places, axes, rot_dim, interleaved, freq, mag):
    """x [heads][hd] float64 of a row whose positions on the axes are places."""
    return ref.turned(x, np.asarray(places)[axes], rot_dim, interleaved, freq, mag)


class Pages:
    """The tables of a cache in pages, one step after another."""

    def __init__(self, sequences, pages, page, max_positions):
        self.page, self.max_positions = page, max_positions
        self.lists = [[] for _ in range(sequences)]
        self.pages = pages

    def refs(self):
        n = [0] * self.pages
        for held in self.lists:
            for p in held:
                n[p] += 1
        return n

    def reach(self, positions):
        return -(-positions // self.page)

    def reserve(self, lens, counts):
        """Returns ok and the copies (sequence, from, to, positions) made."""
        refs, n = self.refs(), len(lens)
        free = [p for p in range(self.pages) if not refs[p]]
        fine = [0 <= s <= len(self.lists[b]) * self.page and s + c <= self.max_positions
                for b, (s, c) in enumerate(zip(lens, counts))]
        slots = [range(lens[b] // self.page, self.reach(lens[b] + counts[b]))
                 if fine[b] and counts[b] else range(0) for b in range(n)]
        writers = {}
        for b in range(n):
            for i in slots[b]:
                if i < len(self.lists[b]) and refs[self.lists[b][i]] > 1:
                    writers.setdefault(self.lists[b][i], []).append(b)
        got, copies, out = [True] * n, [], False
        for b in range(n):
            leave = [i for i in slots[b] if i < len(self.lists[b]) and
                     refs[self.lists[b][i]] > 1 and
                     not (len(writers[self.lists[b][i]]) == refs[self.lists[b][i]] and
                          writers[self.lists[b][i]][0] == b)]
            more = [i for i in slots[b] if i >= len(self.lists[b])]
            if not leave and not more:
                continue
            out = out or len(leave) + len(more) > len(free)
            got[b] = not out
            if out:
                continue
            for i in sorted(leave + more):
                p = free.pop(0)
                if i < len(self.lists[b]):
                    if i == slots[b][0] and lens[b] % self.page:
                        copies.append((b, self.lists[b][i], p, lens[b] % self.page))
                    self.lists[b][i] = p
                else:
                    self.lists[b].append(p)
        refs = self.refs()
        ok = [int(fine[b] and got[b] and
                  not any(refs[self.lists[b][i]] > 1 for i in slots[b] if i < len(self.lists[b])))
              for b in range(n)]
        return ok, copies

    def fork(self, sources, lens):
        was = [list(held) for held in self.lists]
        for b, (s, n) in enumerate(zip(sources, lens)):
            if s == -1:
                self.lists[b] = []
            elif 0 <= s < len(was) and 0 <= n <= len(was[s]) * self.page:
                self.lists[b] = was[s][:self.reach(n)]

    def release(self, lens):
        for b, n in enumerate(lens):
            if n >= 0:
                del self.lists[b][self.reach(n):]

    def compact(self):
        """Returns the number of pages in use and the moves {from: to}."""
        refs = self.refs()
        used = sum(r > 0 for r in refs)
        to = dict(zip([p for p in range(used, self.pages) if refs[p]],
                      [p for p in range(used) if not refs[p]]))
        self.lists = [[to.get(p, p) for p in held] for held in self.lists]
        return used, to

    def table(self):
        most = self.reach(self.max_positions)
        return np.array([held + [-1] * (most - len(held)) for held in self.lists])
