"""What the entry points of caches in pages and of positions on several axes refuse
before anything reaches a device, on the CPU: a program linked to the library with
handles filled in by hand (no device is opened), every call with one argument wrong."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "mormot2-qwen-tts_amd")
HIPCC = "/opt/rocm/bin/hipcc"

SOURCE = r"""
#include <cstdio>
#include <functional>

#include "q3h.h"
#include "q3h_api_internal.h"
#include "q3h_draft.h"

static int bad = 0;
static void expect(const char *what, int want, long long got) {
  if (got != want) {
    std::printf("%s: %lld instead of %d (%s)\n", what, got, want, q3h_last_error());
    bad++;
  } else if (want != 0 && !q3h_last_error()[0]) {
    std::printf("%s: no message\n", what);
    bad++;
  }
}

int main() {
  q3h_device dev, other;
  dev.ordinal = 0;
  other.ordinal = 1;
  static float mem[1 << 12];
  static int32_t ints[4096];
  q3h_cache whole, c;
  whole.dev = c.dev = &dev;
  whole.cfg = c.cfg = {4, 2, 2, 64, 100, Q3H_KV_Q4};
  whole.data = c.data = (char *)mem;
  c.pages = 8, c.page_log2 = 5, c.slots = 4;
  c.state = ints;

  expect("reserve: no cache", Q3H_E_ARG, q3h_cache_reserve(nullptr, 1, 1, ints, ints, ints, 0));
  expect("reserve: no pages", Q3H_E_ARG, q3h_cache_reserve(&whole, 1, 1, ints, ints, ints, 0));
  expect("reserve: sequences", Q3H_E_ARG, q3h_cache_reserve(&c, 5, 1, ints, ints, ints, 0));
  expect("reserve: sequences below 0", Q3H_E_ARG, q3h_cache_reserve(&c, -1, 1, ints, ints, ints, 0));
  expect("reserve: rows below 0", Q3H_E_ARG, q3h_cache_reserve(&c, 1, -1, ints, ints, ints, 0));
  expect("reserve: rows", Q3H_E_CAPACITY, q3h_cache_reserve(&c, 1, 101, ints, ints, ints, 0));
  expect("reserve: lens", Q3H_E_ARG, q3h_cache_reserve(&c, 1, 1, nullptr, ints, ints, 0));
  expect("reserve: nothing to do", Q3H_OK, q3h_cache_reserve(&c, 0, 1, nullptr, ints, ints, 0));
  expect("fork: no cache", Q3H_E_ARG, q3h_cache_fork(nullptr, 1, ints, ints, 0));
  expect("fork: no pages", Q3H_E_ARG, q3h_cache_fork(&whole, 1, ints, ints, 0));
  expect("fork: sequences", Q3H_E_ARG, q3h_cache_fork(&c, 5, ints, ints, 0));
  expect("fork: sources", Q3H_E_ARG, q3h_cache_fork(&c, 1, nullptr, ints, 0));
  expect("fork: lens", Q3H_E_ARG, q3h_cache_fork(&c, 1, ints, nullptr, 0));
  expect("fork: nothing to do", Q3H_OK, q3h_cache_fork(&c, 0, nullptr, nullptr, 0));
  expect("release: no cache", Q3H_E_ARG, q3h_cache_release(nullptr, 1, ints, 0));
  expect("release: no pages", Q3H_E_ARG, q3h_cache_release(&whole, 1, ints, 0));
  expect("release: sequences", Q3H_E_ARG, q3h_cache_release(&c, 5, ints, 0));
  expect("release: lens", Q3H_E_ARG, q3h_cache_release(&c, 1, nullptr, 0));
  expect("compact: no cache", Q3H_E_ARG, q3h_cache_compact(nullptr, ints, 0));
  expect("compact: no pages", Q3H_E_ARG, q3h_cache_compact(&whole, ints, 0));
  expect("state: no cache", Q3H_E_ARG, q3h_cache_page_state(nullptr, ints, ints, ints, 0));
  expect("state: no pages", Q3H_E_ARG, q3h_cache_page_state(&whole, ints, ints, ints, 0));
  expect("state: nothing", Q3H_OK, q3h_cache_page_state(&c, nullptr, nullptr, nullptr, 0));

  // copies
  auto copy = [&](const char *what, int want, std::function<void(q3h_cache &)> edit, int n = 1) {
    q3h_cache from = whole;
    edit(from);
    expect(what, want, q3h_cache_copy(&c, &from, n, ints, ints, 0));
  };
  expect("copy: no cache", Q3H_E_ARG, q3h_cache_copy(nullptr, &whole, 1, ints, ints, 0));
  expect("copy: no source", Q3H_E_ARG, q3h_cache_copy(&c, nullptr, 1, ints, ints, 0));
  expect("copy: itself", Q3H_E_ARG, q3h_cache_copy(&c, &c, 1, ints, ints, 0));
  expect("copy: sources", Q3H_E_ARG, q3h_cache_copy(&c, &whole, 1, nullptr, ints, 0));
  expect("copy: lens", Q3H_E_ARG, q3h_cache_copy(&c, &whole, 1, ints, nullptr, 0));
  copy("copy: sequences", Q3H_E_ARG, [](auto &) {}, 5);
  copy("copy: format", Q3H_E_ARG, [](auto &s) { s.cfg.format = Q3H_KV_Q8; });
  copy("copy: layers", Q3H_E_ARG, [](auto &s) { s.cfg.layers = 3; });
  copy("copy: heads", Q3H_E_ARG, [](auto &s) { s.cfg.kv_heads = 1; });
  copy("copy: head_dim", Q3H_E_ARG, [](auto &s) { s.cfg.head_dim = 128; });
  copy("copy: device", Q3H_E_ARG, [&](auto &s) { s.dev = &other; });
  copy("copy: nothing to do", Q3H_OK, [](auto &) {}, 0);

  // positions on axes
  q3h_rope rope;
  rope.dev = &dev;
  rope.cfg.head_dim = rope.cfg.rot_dim = 64;
  rope.cfg.max_positions = 100;
  q3h_append_args a{};
  a.layer = 1, a.sequences = 4, a.rows = 10;
  a.k = a.v = mem, a.ldk = a.ldv = 128;
  a.lens = ints;
  a.rope = &rope;
  expect("append at: no cache", Q3H_E_ARG, q3h_cache_append_at(nullptr, &a, ints, 0));
  expect("append at: no arguments", Q3H_E_ARG, q3h_cache_append_at(&c, nullptr, ints, 0));
  expect("append at: positions", Q3H_E_ARG, q3h_cache_append_at(&c, &a, nullptr, 0));
  q3h_append_args b = a;
  b.rope = nullptr;
  expect("append at: rope", Q3H_E_ARG, q3h_cache_append_at(&c, &b, ints, 0));
  b = a;
  b.rows = 101;
  expect("append at: rows", Q3H_E_CAPACITY, q3h_cache_append_at(&c, &b, ints, 0));
  b = a;
  b.rows = 0;
  expect("append at: nothing to do", Q3H_OK, q3h_cache_append_at(&c, &b, ints, 0));
  q3h_rope_config r{};
  r.head_dim = r.rot_dim = 64, r.max_positions = 10, r.theta = 1e4f;
  q3h_rope *ro = nullptr;
  int32_t axes[32] = {};
  expect("rope axes: none", Q3H_E_ARG, q3h_rope_create_axes(&dev, &r, 3, nullptr, &ro));
  expect("rope axes: 0", Q3H_E_ARG, q3h_rope_create_axes(&dev, &r, 0, axes, &ro));
  expect("rope axes: 5", Q3H_E_ARG, q3h_rope_create_axes(&dev, &r, 5, axes, &ro));
  axes[31] = 3;
  expect("rope axes: beyond", Q3H_E_ARG, q3h_rope_create_axes(&dev, &r, 3, axes, &ro));
  axes[31] = -1;
  expect("rope axes: below 0", Q3H_E_ARG, q3h_rope_create_axes(&dev, &r, 3, axes, &ro));
  expect("rope axes: no device", Q3H_E_ARG, q3h_rope_create_axes(nullptr, &r, 3, axes, &ro));

  // handles
  q3h_cache *co = nullptr;
  auto cache = [&](const char *what, std::function<void(q3h_paged_config &)> edit) {
    q3h_paged_config p{{2, 1, 2, 64, 100, Q3H_KV_Q4}, 10, 32};
    edit(p);
    expect(what, Q3H_E_ARG, q3h_cache_create_paged(&dev, &p, &co));
  };
  expect("cache: no config", Q3H_E_ARG, q3h_cache_create_paged(&dev, nullptr, &co));
  cache("cache: sequences", [](auto &p) { p.cache.sequences = 0; });
  cache("cache: head_dim", [](auto &p) { p.cache.head_dim = 32; });
  cache("cache: format 3", [](auto &p) { p.cache.format = 3; });
  cache("cache: format 5", [](auto &p) { p.cache.format = 5; });
  cache("cache: no pages", [](auto &p) { p.pages = 0; });
  cache("cache: too many pages", [](auto &p) { p.pages = Q3H_MAX_PAGES + 1; });
  for (int positions : {0, 16, 48, 512, -32})
    cache("cache: page_positions", [&](auto &p) { p.page_positions = positions; });
  cache("cache: too many slots", [](auto &p) {
    p.cache.sequences = 65535;
    p.cache.max_positions = 1 << 14;
  });

  // the workspace of even shares grows with nothing but the heads' size
  c.cfg.max_positions = 1 << 20;
  const int64_t some = q3h_cache_attend_workspace(&c, 1, 1, 4, 1 << 19);
  const int64_t more = q3h_cache_attend_workspace(&c, 4, 4, 8, 1 << 19);
  if (some <= 0 || more < some || more > (16 << 20)) {
    std::printf("workspaces of %lld and %lld bytes\n", (long long)some, (long long)more);
    bad++;
  }
  std::printf("%d wrong\n", bad);
  return bad != 0;
}
"""


def test_host_checks(tmp_path, q3h):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    src, exe = str(tmp_path / "refusals.hip"), str(tmp_path / "refusals")
    with open(src, "w") as f:
        f.write(SOURCE)
    subprocess.run([HIPCC, "-O1", "-std=c++17", "--offload-host-only", "-I",
                    os.path.join(ROOT, "include"), "-I", os.path.join(PKG, "csrc"), src,
                    "-L" + PKG, "-l:libq3h.so", "-Wl,-rpath," + PKG, "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


def test_the_model_of_the_tables():
    """The lists that the device's tables are tested against, on a history by hand."""
    import pages_ref as pref
    m = pref.Pages(3, 6, 32, 100)
    assert m.reserve([0, 0, 0], [40, 10, 0]) == ([1, 1, 1], [])
    assert m.lists == [[0, 1], [2], []]
    m.fork([0, 0, 0], [40, 33, 32])
    assert m.lists == [[0, 1], [0, 1], [0]] and m.refs() == [3, 2, 0, 0, 0, 0]
    # both that hold page 1 write to it: the first keeps it, the other copies one row
    assert m.reserve([40, 33, 32], [1, 1, 1]) == ([1, 1, 1], [(1, 1, 2, 1)])
    assert m.lists == [[0, 1], [0, 2], [0, 3]]
    # page 0 is everyone's: one that writes to it leaves it
    ok, copies = m.reserve([0, 70, 0], [5, 5, 0])
    assert ok == [1, 0, 1] and copies == [] and m.lists[0] == [4, 1]
    m.release([0, 33, 10])
    assert m.lists == [[], [0, 2], [0]]
    assert m.compact() == (2, {2: 1}) and m.lists == [[], [0, 1], [0]]
    # too few: none for the one that asks for too many, nor for who comes after it (whose
    # row would go to page 0, which the other holds too)
    ok, _ = m.reserve([0, 33, 10], [100, 40, 1])
    assert ok == [1, 0, 0] and m.lists == [[2, 3, 4, 5], [0, 1], [0]]
