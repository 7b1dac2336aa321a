"""What the host works out before rows of drafts are launched - the room of a
forward's buffers, counts that a launch or 32 bits hold - on the CPU: a program
linked to the library with handles filled in by hand (no device is opened)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "mormot2-qwen-tts_amd")
HIPCC = "/opt/rocm/bin/hipcc"

HEAD = r"""
#include <algorithm>
#include <cstdio>
#include <initializer_list>

#include "q3h.h"
#include "q3h_api_internal.h"
#include "q3h_draft.h"

static int bad = 0;
#define EXPECT(x, ...)                    \
  do {                                    \
    if (!(x)) {                           \
      std::printf("%s: ", #x);            \
      std::printf(__VA_ARGS__);           \
      std::printf("\n");                  \
      bad++;                              \
    }                                     \
  } while (0)

// 16 heads over 8 of 128, the layers' widths those of a small talker
static void dims(q3h_stack &s, int fmt, int max_positions) {
  s.cfg.layers = 2, s.cfg.hidden = 1024, s.cfg.heads = 16, s.cfg.kv_heads = 8;
  s.cfg.head_dim = 128, s.cfg.intermediate = 2048, s.cfg.kv_f16 = fmt;
  s.cfg.max_positions = max_positions;
  s.ext = true;
}
"""


def run(tmp_path, body):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    src, exe = str(tmp_path / "limits.hip"), str(tmp_path / "limits")
    with open(src, "w") as f:
        f.write(HEAD + "int main() {" + body +
                'std::printf("%d wrong\\n", bad); return bad != 0; }\n')
    subprocess.run([HIPCC, "-O1", "-std=c++17", "--offload-host-only", "-I",
                    os.path.join(ROOT, "include"), "-I", os.path.join(PKG, "csrc"), src,
                    "-L" + PKG, "-l:libq3h.so", "-Wl,-rpath," + PKG, "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


def test_forwards_without_allocations_fit(tmp_path, q3h):
    """Every call of up to 64 rows on a stack whose attention leaves parts fits the
    array at every length, a single row with all the parts that it asks for; the
    parts end within the array and begin behind the other buffers."""
    run(tmp_path, r"""
  static char mem[1];
  for (int fmt : {Q3H_KV_F32, Q3H_KV_Q8})
    for (int head : {0, 2048, 4096}) {
      q3h_stack s;
      dims(s, fmt, 32768);
      for (int rows = 1; rows <= Q3H_NOALLOC_MAX_ROWS; rows++) {
        q3h::Work none;
        const bool fits = q3h::work_carve(&s, rows, 0, head, 0, mem, Q3H_NOALLOC_SCRATCH_BYTES, none);
        EXPECT(fits, "%d rows without parts", rows);
        for (int len : {0, 100, 200, 390, 550, 1000, 3000, 10000, 32768 - rows}) {
          const size_t want = q3h::tree_bytes(&s, 1, rows, len + rows);
          q3h::Work w;
          EXPECT(q3h::work_carve(&s, rows, 0, head, want, mem, Q3H_NOALLOC_SCRATCH_BYTES, w),
                 "%d rows after %d, format %d, head %d", rows, len, fmt, head);
          const char *at = (const char *)w.tree;
          EXPECT(w.tree_bytes <= want && (rows > 1 || w.tree_bytes == want), "%d rows after %d: %zu of %zu",
                 rows, len, w.tree_bytes, want);
          EXPECT(w.tree_bytes == 0 || (at > (char *)w.gpart && at + w.tree_bytes <= mem + Q3H_NOALLOC_SCRATCH_BYTES &&
                                       (at - mem) % 256 == 0), "%d rows after %d", rows, len);
          EXPECT(want == 0 || w.tree_bytes > 0, "%d rows after %d: no parts", rows, len);
        }
      }
    }
""")


def test_counts_of_a_forward_beyond_32_bits_are_refused(tmp_path, q3h):
    """Where a forward's buffers are sized, as q3h_cache_attend refuses its own; the
    largest that a stack of 32 heads over 8 takes is not refused."""
    run(tmp_path, r"""
  auto code = [](const q3h_stack &s, int n, int rows, int positions, bool drafted) {
    try {
      q3h::tree_bytes(&s, n, rows, positions, drafted);
    } catch (const q3h::Error &e) {
      return e.code;
    }
    return 0;
  };
  q3h_stack s;
  dims(s, Q3H_KV_Q8, 65536);
  s.cfg.heads = 32;
  EXPECT(code(s, 1, 65536, 65536, false) == 0, "a prompt of all positions");
  EXPECT(code(s, 256, 1, 65536, false) == 0, "a batch");
  s.cfg.heads = 4096, s.cfg.kv_heads = 1024;
  EXPECT(code(s, 1, 65536, 65536, false) == Q3H_E_CAPACITY, "a prompt over 1024 heads");
  EXPECT(code(s, 65536, 1, 65536, false) == Q3H_E_CAPACITY, "a batch over 1024 heads");
  s.ext = false;
  s.cfg.kv_f16 = Q3H_KV_F16;
  EXPECT(code(s, 65536, 64, 65536, true) == Q3H_E_CAPACITY, "trees");
  EXPECT(code(s, 65536, 64, 65536, false) == 0, "no attention over drafted rows");
""")


def test_scores_of_more_rows_than_a_launch_takes_are_refused(tmp_path, q3h):
    """2^24 workgroups, several for each row of a large vocabulary."""
    run(tmp_path, r"""
  q3h_device dev;
  dev.ordinal = 0;
  alignas(256) static float mem[64];
  static int32_t ints[1];
  for (int vocab : {100, 10234, 151936, 1 << 20}) {
    const int per_row = vocab + 7 <= 10240 ? 1 : (vocab + 7 + 10239) / 10240;
    for (int rows : {((1 << 24) + per_row - 1) / per_row, 1 << 24, 2147483647}) {
      q3h_score_args a{};
      a.logits = mem, a.ld = vocab, a.dtype = Q3H_BF16, a.rows = rows, a.vocab = vocab;
      a.tokens_per_row = 1, a.tokens = ints, a.logprobs = mem;
      a.workspace = mem, a.workspace_bytes = INT64_MAX;
      const int rc = q3h_token_logprobs(&dev, &a, nullptr);
      EXPECT(rc == Q3H_E_CAPACITY, "%d rows of %d: %d (%s)", rows, vocab, rc, q3h_last_error());
      const long long need = q3h_token_logprobs_workspace(rows, vocab, 0);
      EXPECT(need == Q3H_E_CAPACITY, "workspace of %d rows of %d: %lld", rows, vocab, need);
    }
    const int most = ((1 << 24) - 1) / per_row;
    EXPECT(q3h_token_logprobs_workspace(most, vocab, 0) >= 0, "workspace of %d rows of %d", most, vocab);
  }
""")
