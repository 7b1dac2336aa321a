"""What the entry points of drafted rows refuse before anything reaches a
device, on the CPU: a program linked to the library with handles filled in by
hand (no device is opened), every call with one argument wrong. Nothing here
launches: a call that passed its checks would fail for want of a device, with
another code."""
import os
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "mormot2-qwen-tts_amd")
HIPCC = "/opt/rocm/bin/hipcc"

SOURCE = r"""
#include <cmath>
#include <cstddef>
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
  // what the binding packs
  std::printf("sizes %zu %zu %zu %zu %zu %zu\n", sizeof(q3h_append_args),
              offsetof(q3h_append_args, rope), sizeof(q3h_attend_args),
              offsetof(q3h_attend_args, lens), sizeof(q3h_score_args),
              offsetof(q3h_score_args, tokens));
  q3h_device dev, other;
  dev.ordinal = 0;
  other.ordinal = 1;
  q3h_cache c;
  c.dev = &dev;
  c.cfg = {4, 2, 2, 64, 100, Q3H_KV_Q8};
  alignas(256) static float mem[1 << 16];
  c.data = (char *)mem;
  static int32_t ints[4096];
  q3h_rope rope;
  rope.dev = &dev;
  rope.cfg.head_dim = 64;
  rope.cfg.rot_dim = 64;
  rope.cfg.max_positions = 100;

  // more than a launch or 32-bit counts hold
  {
    q3h_cache wide = c;
    wide.cfg = {65535, 1, 1024, 64, 1 << 24, Q3H_KV_Q8};
    q3h_append_args a{};
    a.sequences = 65535, a.rows = 257;
    a.k = a.v = mem, a.lens = ints;
    a.ldk = a.ldv = 65536;
    expect("append: 2^24 rows", Q3H_E_CAPACITY, q3h_cache_append(&wide, &a, nullptr));
    expect("read: 2^32 threads", Q3H_E_CAPACITY,
           q3h_cache_read(&wide, 0, 65535, 9, ints, ints, mem, mem, nullptr));
    for (int rows : {1, 100, 1 << 20, 1 << 24})
      for (int heads : {1024, 4096})
        for (int len : {100, 1 << 24}) {
          q3h_attend_args t{};
          t.sequences = 65535, t.rows = rows, t.heads = heads, t.max_len = len;
          t.q = mem, t.ldq = 64 * heads, t.out = mem + 64, t.ld_out = 64 * heads;
          t.lens = ints;
          expect("attend: 2^32 threads", Q3H_E_CAPACITY, q3h_cache_attend(&wide, &t, nullptr));
          expect("workspace: 2^32 threads", Q3H_E_CAPACITY,
                 q3h_cache_attend_workspace(&wide, 65535, rows, heads, len));
        }
    // one long prompt of many heads, as far as the counts go
    wide.cfg = {1, 1, 1, 128, 1 << 24, Q3H_KV_F16};
    expect("workspace: a prompt of 2^24", Q3H_E_CAPACITY,
           q3h_cache_attend_workspace(&wide, 1, 1 << 24, 64, 0));
    if (q3h_cache_attend_workspace(&wide, 1, 1 << 16, 64, 1 << 10) <= 0) {
      std::printf("workspace: a prompt of 2^16: %s\n", q3h_last_error());
      bad++;
    }
  }

  // append
  q3h_append_args a{};
  a.layer = 1, a.sequences = 4, a.rows = 10, a.heads = 4;
  a.q = a.k = a.v = mem;
  a.ldq = 256, a.ldk = a.ldv = 128;
  a.q_out = mem + 1024, a.ld_out = 256;
  a.lens = ints;
  a.rope = &rope;
  auto append = [&](const char *what, int want, std::function<void(q3h_append_args &)> edit) {
    q3h_append_args b = a;
    edit(b);
    expect(what, want, q3h_cache_append(&c, &b, nullptr));
  };
  expect("append: no cache", Q3H_E_ARG, q3h_cache_append(nullptr, &a, nullptr));
  expect("append: no arguments", Q3H_E_ARG, q3h_cache_append(&c, nullptr, nullptr));
  append("append: layer", Q3H_E_ARG, [](auto &b) { b.layer = 2; });
  append("append: layer below 0", Q3H_E_ARG, [](auto &b) { b.layer = -1; });
  append("append: sequences", Q3H_E_ARG, [](auto &b) { b.sequences = 5; });
  append("append: sequences below 0", Q3H_E_ARG, [](auto &b) { b.sequences = -1; });
  append("append: rows below 0", Q3H_E_ARG, [](auto &b) { b.rows = -1; });
  append("append: rows beyond the cache", Q3H_E_CAPACITY, [](auto &b) { b.rows = 101; });
  append("append: heads below 0", Q3H_E_ARG, [](auto &b) { b.heads = -1; });
  append("append: k", Q3H_E_ARG, [](auto &b) { b.k = nullptr; });
  append("append: v", Q3H_E_ARG, [](auto &b) { b.v = nullptr; });
  append("append: lens", Q3H_E_ARG, [](auto &b) { b.lens = nullptr; });
  append("append: q", Q3H_E_ARG, [](auto &b) { b.q = nullptr; });
  append("append: q_out", Q3H_E_ARG, [](auto &b) { b.q_out = nullptr; });
  append("append: ldq", Q3H_E_ARG, [](auto &b) { b.ldq = 255; });
  append("append: ldk", Q3H_E_ARG, [](auto &b) { b.ldk = 127; });
  append("append: ldv", Q3H_E_ARG, [](auto &b) { b.ldv = 127; });
  append("append: ld_out", Q3H_E_ARG, [](auto &b) { b.ld_out = 255; });
  append("append: in place, another distance", Q3H_E_ARG, [](auto &b) {
    b.q_out = const_cast<float *>(b.q);
    b.ld_out = 512;
  });
  append("append: eps", Q3H_E_ARG, [](auto &b) {
    b.k_norm = b.k;
    b.eps = -1.f;
  });
  append("append: tree of 65 rows", Q3H_E_CAPACITY, [](auto &b) {
    b.rows = 65;
    b.parents = ints;
  });
  rope.cfg.max_positions = 99;
  append("append: rope table", Q3H_E_ARG, [](auto &) {});
  rope.cfg.max_positions = 100;
  rope.cfg.head_dim = 128;
  append("append: rope head", Q3H_E_ARG, [](auto &) {});
  rope.cfg.head_dim = 64;
  rope.dev = &other;
  append("append: rope of another device", Q3H_E_ARG, [](auto &) {});
  rope.dev = &dev;
  append("append: nothing to do", Q3H_OK, [](auto &b) { b.rows = 0; });
  append("append: no sequence", Q3H_OK, [](auto &b) { b.sequences = 0; });

  // read
  expect("read: no cache", Q3H_E_ARG, q3h_cache_read(nullptr, 0, 1, 1, ints, ints, mem, mem, 0));
  expect("read: layer", Q3H_E_ARG, q3h_cache_read(&c, 2, 1, 1, ints, ints, mem, mem, 0));
  expect("read: sequences", Q3H_E_ARG, q3h_cache_read(&c, 0, 5, 1, ints, ints, mem, mem, 0));
  expect("read: rows", Q3H_E_CAPACITY, q3h_cache_read(&c, 0, 1, 101, ints, ints, mem, mem, 0));
  expect("read: nothing", Q3H_OK, q3h_cache_read(&c, 0, 1, 1, ints, ints, nullptr, nullptr, 0));

  // attention
  q3h_attend_args t{};
  t.layer = 0, t.sequences = 4, t.rows = 10, t.heads = 4, t.max_len = 90;
  t.q = mem, t.out = mem + 4096, t.ldq = t.ld_out = 256;
  t.lens = ints;
  t.workspace = mem;
  t.workspace_bytes = sizeof(mem);
  auto attend = [&](const char *what, int want, std::function<void(q3h_attend_args &)> edit) {
    q3h_attend_args b = t;
    edit(b);
    expect(what, want, q3h_cache_attend(&c, &b, nullptr));
  };
  expect("attend: no cache", Q3H_E_ARG, q3h_cache_attend(nullptr, &t, nullptr));
  expect("attend: no arguments", Q3H_E_ARG, q3h_cache_attend(&c, nullptr, nullptr));
  attend("attend: layer", Q3H_E_ARG, [](auto &b) { b.layer = 2; });
  attend("attend: sequences", Q3H_E_ARG, [](auto &b) { b.sequences = 5; });
  attend("attend: rows", Q3H_E_CAPACITY, [](auto &b) { b.rows = 101; });
  attend("attend: no heads", Q3H_E_ARG, [](auto &b) { b.heads = 0; });
  attend("attend: heads", Q3H_E_ARG, [](auto &b) { b.heads = 5; });
  attend("attend: max_len", Q3H_E_ARG, [](auto &b) { b.max_len = 101; });
  attend("attend: max_len below 0", Q3H_E_ARG, [](auto &b) { b.max_len = -1; });
  attend("attend: q", Q3H_E_ARG, [](auto &b) { b.q = nullptr; });
  attend("attend: out", Q3H_E_ARG, [](auto &b) { b.out = nullptr; });
  attend("attend: lens", Q3H_E_ARG, [](auto &b) { b.lens = nullptr; });
  attend("attend: ldq", Q3H_E_ARG, [](auto &b) { b.ldq = 255; });
  attend("attend: ld_out", Q3H_E_ARG, [](auto &b) { b.ld_out = 255; });
  attend("attend: in place, another distance", Q3H_E_ARG, [](auto &b) {
    b.out = const_cast<float *>(b.q);
    b.ld_out = 512;
  });
  attend("attend: scale", Q3H_E_ARG, [](auto &b) { b.scale = NAN; });
  attend("attend: tree of 65 rows", Q3H_E_CAPACITY, [](auto &b) {
    b.rows = 65;
    b.parents = ints;
  });
  attend("attend: nothing to do", Q3H_OK, [](auto &b) { b.sequences = 0; });
  // a long context of one row is split, its parts in the workspace
  c.cfg.max_positions = 1 << 20;
  const int64_t need = q3h_cache_attend_workspace(&c, 1, 1, 4, 1 << 19);
  if (need > 0) {
    auto longer = [&](q3h_attend_args &b) {
      b.sequences = b.rows = 1;
      b.max_len = 1 << 19;
    };
    attend("attend: no workspace", Q3H_E_ARG, [&](auto &b) {
      longer(b);
      b.workspace = nullptr;
    });
    attend("attend: a small workspace", Q3H_E_ARG, [&](auto &b) {
      longer(b);
      b.workspace_bytes = need - 1;
    });
    attend("attend: an odd workspace", Q3H_E_ARG, [&](auto &b) {
      longer(b);
      b.workspace = (char *)mem + 64;
      b.workspace_bytes = need;
    });
  }
  c.cfg.max_positions = 100;
  expect("workspace: heads", Q3H_E_ARG, q3h_cache_attend_workspace(&c, 1, 1, 3, 10));
  expect("workspace: max_len", Q3H_E_ARG, q3h_cache_attend_workspace(&c, 1, 1, 4, 101));
  expect("workspace: no cache", Q3H_E_ARG, q3h_cache_attend_workspace(nullptr, 1, 1, 4, 10));

  // keep
  expect("keep: no cache", Q3H_E_ARG, q3h_cache_keep(nullptr, 1, 1, ints, ints, ints, 0));
  expect("keep: lens", Q3H_E_ARG, q3h_cache_keep(&c, 1, 1, nullptr, ints, ints, 0));
  expect("keep: kept", Q3H_E_ARG, q3h_cache_keep(&c, 1, 1, ints, nullptr, ints, 0));
  expect("keep: counts", Q3H_E_ARG, q3h_cache_keep(&c, 1, 1, ints, ints, nullptr, 0));
  expect("keep: sequences", Q3H_E_ARG, q3h_cache_keep(&c, 5, 1, ints, ints, ints, 0));
  expect("keep: rows", Q3H_E_CAPACITY, q3h_cache_keep(&c, 1, 101, ints, ints, ints, 0));

  // scores
  q3h_score_args s{};
  s.logits = mem, s.ld = 500, s.dtype = Q3H_F32, s.rows = 3, s.vocab = 500;
  s.tokens_per_row = 2, s.top_k = 4, s.tokens = ints;
  s.logprobs = mem, s.entropy = mem, s.top_ids = ints, s.top_logprobs = mem;
  s.workspace = mem, s.workspace_bytes = sizeof(mem);
  auto score = [&](const char *what, int want, std::function<void(q3h_score_args &)> edit) {
    q3h_score_args b = s;
    edit(b);
    expect(what, want, q3h_token_logprobs(&dev, &b, nullptr));
  };
  expect("score: no device", Q3H_E_ARG, q3h_token_logprobs(nullptr, &s, nullptr));
  expect("score: no arguments", Q3H_E_ARG, q3h_token_logprobs(&dev, nullptr, nullptr));
  score("score: rows", Q3H_E_ARG, [](auto &b) { b.rows = -1; });
  score("score: vocab", Q3H_E_ARG, [](auto &b) { b.vocab = 0; });
  score("score: dtype", Q3H_E_ARG, [](auto &b) { b.dtype = Q3H_Q8_0; });
  score("score: tokens_per_row", Q3H_E_ARG, [](auto &b) { b.tokens_per_row = -1; });
  score("score: top_k", Q3H_E_ARG, [](auto &b) { b.top_k = 65; });
  score("score: top_k beyond vocab", Q3H_E_ARG, [](auto &b) { b.vocab = 3; });
  score("score: logits", Q3H_E_ARG, [](auto &b) { b.logits = nullptr; });
  score("score: ld", Q3H_E_ARG, [](auto &b) { b.ld = 499; });
  score("score: tokens", Q3H_E_ARG, [](auto &b) { b.tokens = nullptr; });
  score("score: logprobs", Q3H_E_ARG, [](auto &b) { b.logprobs = nullptr; });
  score("score: top_ids", Q3H_E_ARG, [](auto &b) { b.top_ids = nullptr; });
  score("score: top_logprobs", Q3H_E_ARG, [](auto &b) { b.top_logprobs = nullptr; });
  score("score: nothing to do", Q3H_OK, [](auto &b) { b.rows = 0; });
  const int64_t room = q3h_token_logprobs_workspace(1, 1 << 20, 4);
  if (room > 0)
    score("score: no workspace", Q3H_E_ARG, [](auto &b) {
      b.rows = 1;
      b.ld = b.vocab = 1 << 20;
      b.workspace = nullptr;
    });
  expect("score workspace: top_k", Q3H_E_ARG, q3h_token_logprobs_workspace(1, 10, 11));
  expect("score workspace: rows", Q3H_E_ARG, q3h_token_logprobs_workspace(-1, 10, 1));

  // handles
  q3h_rope_config r{};
  r.head_dim = 64, r.rot_dim = 64, r.max_positions = 10, r.theta = 1e4f, r.factor = 2.f;
  r.original_positions = 100, r.beta_fast = 32.f, r.beta_slow = 1.f, r.low_turns = 1.f;
  r.high_turns = 4.f;
  q3h_rope *ro = nullptr;
  auto table = [&](const char *what, std::function<void(q3h_rope_config &)> edit) {
    q3h_rope_config b = r;
    edit(b);
    expect(what, Q3H_E_ARG, q3h_rope_create(&dev, &b, &ro));
  };
  expect("rope: no device", Q3H_E_ARG, q3h_rope_create(nullptr, &r, &ro));
  expect("rope: no config", Q3H_E_ARG, q3h_rope_create(&dev, nullptr, &ro));
  expect("rope: no out", Q3H_E_ARG, q3h_rope_create(&dev, &r, nullptr));
  table("rope: head_dim", [](auto &b) { b.head_dim = 96; });
  table("rope: rot_dim odd", [](auto &b) { b.rot_dim = 33; });
  table("rope: rot_dim 0", [](auto &b) { b.rot_dim = 0; });
  table("rope: rot_dim above", [](auto &b) { b.rot_dim = 66; });
  table("rope: interleaved", [](auto &b) { b.interleaved = 2; });
  table("rope: positions", [](auto &b) { b.max_positions = 0; });
  table("rope: theta", [](auto &b) { b.theta = 1.f; });
  table("rope: scaling", [](auto &b) { b.scaling = 4; });
  table("rope: factor", [](auto &b) { b.scaling = Q3H_ROPE_LINEAR, b.factor = 0.f; });
  table("rope: span", [](auto &b) { b.scaling = Q3H_ROPE_YARN, b.original_positions = 0; });
  table("rope: betas", [](auto &b) { b.scaling = Q3H_ROPE_YARN, b.beta_slow = 32.f; });
  table("rope: turns", [](auto &b) { b.scaling = Q3H_ROPE_BANDS, b.high_turns = 1.f; });
  table("rope: magnitude", [](auto &b) { b.magnitude = -1.f; });
  table("rope: magnitude NaN", [](auto &b) { b.magnitude = NAN; });
  q3h_cache *co = nullptr;
  auto cache = [&](const char *what, std::function<void(q3h_cache_config &)> edit) {
    q3h_cache_config b{2, 1, 2, 64, 100, Q3H_KV_F32};
    edit(b);
    expect(what, Q3H_E_ARG, q3h_cache_create(&dev, &b, &co));
  };
  expect("cache: no config", Q3H_E_ARG, q3h_cache_create(&dev, nullptr, &co));
  cache("cache: sequences", [](auto &b) { b.sequences = 0; });
  cache("cache: layers", [](auto &b) { b.layers = 0; });
  cache("cache: kv_heads", [](auto &b) { b.kv_heads = -1; });
  cache("cache: head_dim", [](auto &b) { b.head_dim = 32; });
  cache("cache: positions", [](auto &b) { b.max_positions = 0; });
  cache("cache: too many positions", [](auto &b) { b.max_positions = (1 << 24) + 1; });
  cache("cache: format", [](auto &b) { b.format = 3; });
  expect("cache: destroy", Q3H_E_ARG, q3h_cache_destroy(nullptr));
  expect("rope: destroy", Q3H_E_ARG, q3h_rope_destroy(nullptr));
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
    # the binding's formats have the header's sizes and places
    sizes = [int(x) for x in r.stdout.split("\n")[0].split()[1:]]
    assert sizes == [q3h.APPEND_ARGS.size, struct.calcsize("4i3P3qPqPPf0P"),
                     q3h.ATTEND_ARGS.size, struct.calcsize("5ifPqPq"),
                     q3h.SCORE_ARGS.size, struct.calcsize("Pq5i0P")]
