"""Appends by positions on several axes, on the CPU: what they refuse and take, by a program
linked to the library with handles filled in by hand (no device is opened)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "mormot2-qwen-tts_amd")
HIPCC = "/opt/rocm/bin/hipcc"

BEGIN = r"""
#include <cstdio>
#include <cstring>
#include <functional>

#include "q3h.h"
#include "q3h_api_internal.h"
#include "q3h_draft.h"

static int bad = 0;
// want: the code; a refusal's text begins with the call's name
static void expect(const char *what, const char *call, int want, int got) {
  const char *text = q3h_last_error();
  const size_t n = std::strlen(call);
  if (got != want || (want != 0 && (std::strncmp(text, call, n) != 0 || text[n] != ':'))) {
    std::printf("%s: %d instead of %d (%s)\n", what, got, want, text);
    bad++;
  }
}

int main() {
  q3h_device dev, other;
  dev.ordinal = 0;
  other.ordinal = 1;
  static float mem[1 << 12];
  static int32_t ints[4096];
  q3h_cache c;
  c.dev = &dev;
  c.cfg = {4, 2, 2, 64, 100, Q3H_KV_Q4};
  c.data = (char *)mem;
  q3h_rope rope;
  rope.dev = &dev;
  rope.cfg.head_dim = rope.cfg.rot_dim = 64;
  rope.cfg.max_positions = 100;
  q3h_append_args good{};
  good.layer = 1, good.sequences = 4, good.rows = 10, good.heads = 4;
  good.q = good.k = good.v = mem, good.q_out = mem + 64;
  good.ldq = good.ld_out = 256, good.ldk = good.ldv = 128;
  good.lens = ints;
  good.rope = &rope;

  const char *at = "q3h_cache_append_at", *plain = "q3h_cache_append";
"""

END = r"""
  std::printf("%d wrong\n", bad);
  return bad != 0;
}
"""

PARTS = {
    # a refusal names the call that it is of
    "texts": r"""
  // one argument wrong, by both calls
  auto both = [&](const char *what, int want, std::function<void(q3h_append_args &)> edit) {
    q3h_append_args a = good;
    edit(a);
    expect(what, at, want, q3h_cache_append_at(&c, &a, ints, 0));
    expect(what, plain, want, q3h_cache_append(&c, &a, 0));
  };
  both("layer", Q3H_E_ARG, [](auto &a) { a.layer = 2; });
  both("sequences", Q3H_E_ARG, [](auto &a) { a.sequences = 5; });
  both("rows", Q3H_E_CAPACITY, [](auto &a) { a.rows = 101; });
  both("heads", Q3H_E_ARG, [](auto &a) { a.heads = -1; });
  both("keys", Q3H_E_ARG, [](auto &a) { a.k = nullptr; });
  both("queries", Q3H_E_ARG, [](auto &a) { a.q_out = nullptr; });
  both("distances", Q3H_E_ARG, [](auto &a) { a.ldk = 127; });
  both("in place", Q3H_E_ARG, [](auto &a) { a.q_out = const_cast<float *>(a.q), a.ldq = 300; });
  both("eps", Q3H_E_ARG, [](auto &a) { a.q_norm = a.q, a.eps = -1.f; });
  both("tree", Q3H_E_CAPACITY, [](auto &a) { a.parents = a.lens, a.rows = 65; });
  rope.dev = &other;
  both("rope's device", Q3H_E_ARG, [](auto &) {});
  rope.dev = &dev;
  rope.cfg.head_dim = 128;
  both("rope's head_dim", Q3H_E_ARG, [](auto &) {});
  rope.cfg.head_dim = 64;
  rope.cfg.max_positions = 99;
  both("rope's positions", Q3H_E_ARG, [](auto &) {});
  rope.cfg.max_positions = 100;
  expect("no cache", at, Q3H_E_ARG, q3h_cache_append_at(nullptr, &good, ints, 0));
  expect("no cache", plain, Q3H_E_ARG, q3h_cache_append(nullptr, &good, 0));
  expect("no arguments", at, Q3H_E_ARG, q3h_cache_append_at(&c, nullptr, ints, 0));
  expect("no arguments or positions", at, Q3H_E_ARG, q3h_cache_append_at(&c, nullptr, nullptr, 0));
  expect("no positions", at, Q3H_E_ARG, q3h_cache_append_at(&c, &good, nullptr, 0));
  q3h_append_args a = good;
  a.rope = nullptr;
  expect("no rope", at, Q3H_E_ARG, q3h_cache_append_at(&c, &a, ints, 0));

  // rotary tables
  q3h_rope_config r{};
  r.head_dim = r.rot_dim = 64, r.max_positions = 10, r.theta = 1e4f;
  q3h_rope *ro = nullptr;
  int32_t axes[32] = {};
  auto tables = [&](const char *what, std::function<void(q3h_rope_config &)> edit) {
    q3h_rope_config x = r;
    edit(x);
    expect(what, "q3h_rope_create", Q3H_E_ARG, q3h_rope_create(&dev, &x, &ro));
    expect(what, "q3h_rope_create_axes", Q3H_E_ARG, q3h_rope_create_axes(&dev, &x, 3, axes, &ro));
  };
  tables("head_dim", [](auto &x) { x.head_dim = 32; });
  tables("rot_dim", [](auto &x) { x.rot_dim = 66; });
  tables("interleaved", [](auto &x) { x.interleaved = 2; });
  tables("max_positions", [](auto &x) { x.max_positions = 0; });
  tables("theta", [](auto &x) { x.theta = 1.f; });
  tables("scaling", [](auto &x) { x.scaling = 4; });
  tables("factor", [](auto &x) { x.scaling = Q3H_ROPE_LINEAR, x.factor = 0.f; });
  tables("magnitude", [](auto &x) { x.magnitude = -1.f; });
  expect("no device", "q3h_rope_create_axes", Q3H_E_ARG,
         q3h_rope_create_axes(nullptr, &r, 3, axes, &ro));
  expect("no config", "q3h_rope_create", Q3H_E_ARG, q3h_rope_create(&dev, nullptr, &ro));
  expect("axes", "q3h_rope_create_axes", Q3H_E_ARG, q3h_rope_create_axes(&dev, &r, 5, axes, &ro));
""",
    # nothing to write: as q3h_cache_append takes it, without positions
    "nothing to write": r"""
  q3h_append_args a = good;
  a.rows = 0;
  a.q = a.k = a.v = nullptr, a.q_out = nullptr, a.lens = nullptr;
  expect("no rows", at, Q3H_OK, q3h_cache_append_at(&c, &a, nullptr, 0));
  expect("no rows", plain, Q3H_OK, q3h_cache_append(&c, &a, 0));
  a.rope = nullptr;
  expect("no rows or rope", at, Q3H_OK, q3h_cache_append_at(&c, &a, nullptr, 0));
  a.rows = 10, a.sequences = 0;
  expect("no sequences", at, Q3H_OK, q3h_cache_append_at(&c, &a, nullptr, 0));
  a.layer = 2;
  expect("no sequences of no layer", at, Q3H_E_ARG, q3h_cache_append_at(&c, &a, nullptr, 0));
""",
}


@pytest.mark.parametrize("part", list(PARTS))
def test_host_checks(tmp_path, q3h, part):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    src, exe = str(tmp_path / "calls.hip"), str(tmp_path / "calls")
    with open(src, "w") as f:
        f.write(BEGIN + PARTS[part] + END)
    subprocess.run([HIPCC, "-O1", "-std=c++17", "--offload-host-only", "-I",
                    os.path.join(ROOT, "include"), "-I", os.path.join(PKG, "csrc"), src,
                    "-L" + PKG, "-l:libq3h.so", "-Wl,-rpath," + PKG, "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
