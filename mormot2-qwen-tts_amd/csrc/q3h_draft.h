// q3h_draft.h - the operators around drafted rows: device views and launchers
// shared by their entry points (q3h_cache.hip, q3h_tree.hip, q3h_score.hip) and
// the stacks' forwards.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "q3h.h"
#include "q3h_internal.h"

namespace q3h {

// bytes of one cache element, and whether rows carry a scale
inline size_t kv_elem_bytes(int fmt) { return fmt == Q3H_KV_F32 ? 4 : fmt == Q3H_KV_F16 ? 2 : 1; }
// bytes of one sequence's cache of `layers` layers (keys, values, their scales)
inline size_t kv_bytes(int fmt, int layers, int kvh, int max_pos, int hd) {
  const size_t rows = (size_t)layers * kvh * max_pos;
  return 2 * rows * (hd * kv_elem_bytes(fmt) + (fmt == Q3H_KV_Q8 ? sizeof(float) : 0));
}

// Where the drafted rows' caches are: one allocation of sequences seq_bytes
// apart, lengths in lens; or the contexts of row descriptors (rd: that of a
// sequence's first row, whose pos is the sequence's length; pos < 0: no rows).
struct KvView {
  char *base;
  int64_t seq_bytes;
  const RowDesc *rd;
  const int32_t *lens, *counts;  // counts nullable
  int layers, kvh, max_pos, layer;
  int sequences, rows;
};

// A sequence of a view on the device: its layer's first key, the elements from
// the keys to the values and (int8) from a key's row to its scale.
struct KvSeq {
  char *k0;
  int max_pos, len, count;
};
__device__ __forceinline__ KvSeq kv_sequence(const KvView &v, int b) {
  KvSeq s;
  if (v.rd) {
    const RowDesc d = v.rd[(size_t)b * v.rows];
    s.k0 = reinterpret_cast<char *>(global_ptr(reinterpret_cast<char *>(d.k)));
    s.max_pos = d.max_pos;
    s.len = d.pos;
    s.count = d.pos < 0 ? 0 : v.rows;
  } else {
    s.k0 = v.base + b * v.seq_bytes;
    s.max_pos = v.max_pos;
    s.len = v.lens[b];
    s.count = v.rows;
  }
  if (v.counts) s.count = min(max(v.counts[b], 0), s.count);
  return s;
}
// a byte of the int8 format: the value + 128
__device__ __forceinline__ float kv_byte(uint8_t b) { return (float)((int)b - 128); }
// the row of (part: 0 keys, 1 values; kv head g; position p) in rows of the
// sequence's allocation: elements at row * HD, int8 scales at
// 2 rows_in_all * HD bytes + 4 row
__device__ __forceinline__ int64_t kv_row(const KvView &v, const KvSeq &s, int part, int g, int p) {
  return (((int64_t)part * v.layers + v.layer) * v.kvh + g) * s.max_pos + p;
}
__device__ __forceinline__ float *kv_scales(const KvView &v, const KvSeq &s, int hd) {
  return reinterpret_cast<float *>(s.k0 + 2 * (int64_t)v.layers * v.kvh * s.max_pos * hd);
}

// The paths of a sequence's drafted rows, lane t for row t (at most 64): which
// rows are on row t's path (bit t itself), its depth, and whether the path
// meets a parent that is not below its row or is under -1. Each step doubles
// the part of the path that is known: six for 64 rows. All lanes active.
struct Path {
  uint64_t rows;
  int depth;
  bool bad;
};
__device__ __forceinline__ Path tree_path(const int32_t *parents, int rows) {
  const int lane = threadIdx.x & 63;
  int p = lane < rows ? parents[lane] : -1;
  int bad = p >= lane || p < -1;
  if (bad) p = -1;
  uint64_t m = 1ull << lane;
  int d = p >= 0;
#pragma unroll
  for (int i = 0; i < 6; i++) {
    const int at = p >= 0 ? p : lane;
    const uint64_t m2 = __shfl(m, at);
    const int d2 = __shfl(d, at), b2 = __shfl(bad, at), p2 = __shfl(p, at);
    if (p >= 0) {
      m |= m2;
      d += d2;
      bad |= b2;
      p = p2;
    }
  }
  return {m, d, bad != 0};
}

struct AppendRows {
  KvView kv;
  int heads;  // query heads, 0: none
  const float *q, *k, *v;
  int64_t ldq, ldk, ldv;
  float *q_out;
  int64_t ld_out;
  const float *q_norm, *k_norm;  // nullable
  float eps;
  // rotary table [position][rot_dim / 2] of (cos, sin) in 64 bits, or a stack's in
  // 32; at most one of them
  const double2 *table;
  const float2 *table32;
  int rot_dim, interleaved;
  const int32_t *parents;  // nullable
};
// hd: 64 or 128; fmt: Q3H_KV_*
void launch_cache_append(const AppendRows &a, int hd, int fmt, hipStream_t st);

struct AttendRows {
  KvView kv;
  int heads, max_len;
  float scale;
  const float *q;
  int64_t ldq;
  float *out;
  int64_t ld_out;
  const int32_t *parents;
  float *part;
  size_t room;  // bytes of part: attend_part_bytes, or less (fewer parts then)
};
size_t attend_part_bytes(int sequences, int rows, int heads, int kvh, int hd, int fmt,
                         int max_len);
// whether a call's work can be counted in 32 bits (2^30 tiles of 16 rows)
bool attend_fits(int sequences, int rows, int heads, int kvh, int hd, int fmt, int max_len);
void launch_cache_attend(const AttendRows &a, int hd, int fmt, hipStream_t st);
// kept rows to the front of the drafted ones, every layer of v: kept [sequences][rows],
// v.counts of them
void launch_cache_keep(const KvView &v, const int32_t *kept, int hd, int fmt, hipStream_t st);
// positions [0, len) of an int8 cache of one sequence (k0: its keys, values behind
// them) from or to f32 [layers][kvh][len][hd]
void launch_q8_fill(const float *src, char *k0, bool values, int layers, int kvh, int len, int hd,
                    int max_pos, hipStream_t st);
void launch_q8_read(const char *k0, bool values, int layers, int layer, int kvh, int len, int hd,
                    int max_pos, float *dst, hipStream_t st);

struct ScoreRows {
  const void *logits;
  int64_t ld;
  bool bf16;
  int rows, vocab, tokens_per_row, top_k;
  const int32_t *tokens;
  float *logprobs, *entropy;
  int32_t *top_ids;
  float *top_logprobs;
  void *work;  // score_work_bytes
};
size_t score_work_bytes(int rows, int vocab, int top_k);
void launch_token_scores(const ScoreRows &a, hipStream_t st);

// A caller's device while an entry point that only enqueues on the caller's
// stream has its own current.
class DeviceScope {
 public:
  explicit DeviceScope(int ordinal);
  ~DeviceScope();
  DeviceScope(const DeviceScope &) = delete;
  DeviceScope &operator=(const DeviceScope &) = delete;

 private:
  int before_ = -1;
};

}  // namespace q3h

struct q3h_rope {
  q3h_device *dev = nullptr;
  q3h_rope_config cfg{};
  double2 *table = nullptr;  // [max_positions][rot_dim / 2]
  int64_t bytes = 0;
};

struct q3h_cache {
  q3h_device *dev = nullptr;
  q3h_cache_config cfg{};
  char *data = nullptr;
  size_t seq_bytes = 0;
  int64_t bytes = 0;
};
