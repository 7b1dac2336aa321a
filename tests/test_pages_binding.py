"""The binding's handles of caches and rotary tables, without a device: a library in its place that counts
what it makes and takes back."""
import ctypes
import gc
import types

import pytest


class Library:
    """The entry points that a handle is made and destroyed with."""

    def __init__(self, real):
        self.real, self.made, self.live, self.lacks = real, 0, set(), None

    def __getattr__(self, name):
        if name == self.lacks:
            raise AttributeError(name)
        return getattr(self.real, name)

    def _make(self, dev, cfg, out):
        self.made += 1
        self.live.add(self.made)
        out._obj.value = self.made
        return 0

    q3h_cache_create = q3h_cache_create_paged = q3h_rope_create = _make

    def q3h_rope_create_axes(self, dev, cfg, axes, pairs, out):
        axes = ctypes.c_int(axes).value  # (what reaches it)
        fine = 1 <= axes <= 4 and all(0 <= x < axes for x in pairs)
        return self._make(dev, cfg, out) if fine else -1

    def q3h_cache_destroy(self, h):
        self.live.remove(h.value)
        return 0

    q3h_rope_destroy = q3h_cache_destroy


@pytest.fixture
def library(q3h, monkeypatch):
    made = Library(q3h.lib())
    monkeypatch.setattr(q3h, "lib", lambda: made)
    return made


DEV = types.SimpleNamespace(h=1, ordinal=0)


def test_a_cache_without_pages_has_no_page_size(q3h, library):
    """page_positions says nothing of a cache in one piece, and is not looked at there."""
    cache = q3h.Cache(DEV, 2, 2, 64, 100, page_positions=0)
    assert len(library.live) == 1
    with pytest.raises(q3h.Q3HError) as e:
        cache.page_state()
    assert e.value.code == q3h.E_ARG
    cache.destroy()
    assert not library.live


@pytest.mark.parametrize("pages", [0, 4])
@pytest.mark.parametrize("fails", ["tensors", "entry point"])
def test_a_cache_that_is_not_finished_is_given_back(q3h, library, monkeypatch, pages, fails):
    """Nothing stays with the library where the binding fails before or behind its call."""
    def no_tensors():
        raise ImportError("no tensors")
    if fails == "tensors":
        monkeypatch.setattr(q3h, "_use_torch", no_tensors)
    else:
        library.lacks = "q3h_cache_page_state"
    with pytest.raises((ImportError, AttributeError)):
        q3h.Cache(DEV, 2, 2, 64, 100, pages=pages)
    gc.collect()
    assert not library.live


def test_caches_in_pages_know_their_tables(q3h, library):
    cache = q3h.Cache(DEV, 3, 2, 64, 100, pages=7, page_positions=32)
    assert cache.table_shape == (3, 4) and cache.pages == 7
    del cache
    gc.collect()
    assert library.made == 1 and not library.live


def test_axes_that_there_are_not(q3h, library):
    """An axis outside 0 .. 3 is refused, one that 32 bits would make another of as well."""
    for axis in (-1, 4, 2 ** 31, 2 ** 32, 2 ** 32 + 1, -2 ** 32):
        with pytest.raises(q3h.Q3HError) as e:
            q3h.Rope(DEV, 64, 100, 1e4, axes=[axis] * 32)
        assert e.value.code == q3h.E_ARG
        with pytest.raises(q3h.Q3HError) as e:
            q3h.Rope(DEV, 64, 100, 1e4, axes=[3] * 31 + [axis])
        assert e.value.code == q3h.E_ARG
    assert library.made == 0
    rope = q3h.Rope(DEV, 64, 100, 1e4, axes=[i % 4 for i in range(32)])
    assert rope.axes == 4 and library.made == 1
