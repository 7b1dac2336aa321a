// q3h_draft.h - the operators around drafted rows: device views and launchers
// shared by their entry points (q3h_cache.hip, q3h_tree.hip, q3h_score.hip) and
// the stacks' forwards.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "q3h.h"
#include "q3h_internal.h"

namespace q3h {

inline bool kv_format(int fmt) {
  return fmt == Q3H_KV_F32 || fmt == Q3H_KV_F16 || fmt == Q3H_KV_Q8 || fmt == Q3H_KV_Q4;
}
// bytes of the elements of one cache row (a head's hd elements at a position)
constexpr int kv_row_bytes(int fmt, int hd) {
  return fmt == Q3H_KV_F32 ? 4 * hd : fmt == Q3H_KV_F16 ? 2 * hd : fmt == Q3H_KV_Q8 ? hd : hd / 2;
}
// whether rows have a scale (f32), and a word of their groups' steps
constexpr bool kv_scaled(int fmt) { return fmt == Q3H_KV_Q8 || fmt == Q3H_KV_Q4; }
// bytes of one sequence's cache of `layers` layers: keys and values, their scales, their
// groups' steps
inline size_t kv_bytes(int fmt, int layers, int kvh, int max_pos, int hd) {
  const size_t rows = (size_t)layers * kvh * max_pos;
  return 2 * rows * (kv_row_bytes(fmt, hd) + (kv_scaled(fmt) ? sizeof(float) : 0) +
                     (fmt == Q3H_KV_Q4 ? sizeof(uint32_t) : 0));
}

// F<format, head_dim>::go(args...)
template <template <int, int> class F, class... A>
void by_format(int hd, int fmt, A &&...args) {
  if (hd == 64) {
    if (fmt == Q3H_KV_F32) F<Q3H_KV_F32, 64>::go(args...);
    else if (fmt == Q3H_KV_F16) F<Q3H_KV_F16, 64>::go(args...);
    else if (fmt == Q3H_KV_Q8) F<Q3H_KV_Q8, 64>::go(args...);
    else F<Q3H_KV_Q4, 64>::go(args...);
  } else {
    if (fmt == Q3H_KV_F32) F<Q3H_KV_F32, 128>::go(args...);
    else if (fmt == Q3H_KV_F16) F<Q3H_KV_F16, 128>::go(args...);
    else if (fmt == Q3H_KV_Q8) F<Q3H_KV_Q8, 128>::go(args...);
    else F<Q3H_KV_Q4, 128>::go(args...);
  }
}

// Where the drafted rows' caches are: one allocation of sequences seq_bytes
// apart, lengths in lens; the pages of a cache (table), each a sequence's cache of
// 1 << page_log2 positions, seq_bytes apart; or the contexts of row descriptors (rd:
// that of a sequence's first row, whose pos is the sequence's length; pos < 0: no rows).
struct KvView {
  char *base;
  int64_t seq_bytes;
  const RowDesc *rd;
  const int32_t *lens, *counts;  // counts nullable
  int layers, kvh, max_pos, layer;
  int sequences, rows;
  // pages: [all sequences][slots], those that each sequence holds, and how many
  // sequences hold each page; table null: none
  const int32_t *table, *held, *refs;
  int pages, slots, page_log2;
};

// A sequence of a view on the device: its first layer's first key and the positions
// that it has room for (the distance of its heads, but of pages).
struct KvSeq {
  char *k0;
  int max_pos, len, count;
};
// positions that a sequence's pages reach
__device__ __forceinline__ int kv_room(const KvView &v, int b) {
  return min((int64_t)v.max_pos, (int64_t)v.held[b] << v.page_log2);
}
// slot `at` of a sequence's pages (a table that is rewritten meanwhile leads to no other memory)
__device__ __forceinline__ int kv_page(const KvView &v, int b, int at) {
  const int page = v.table[(size_t)b * v.slots + at];
  return (uint32_t)page < (uint32_t)v.pages ? page : 0;
}
// (PAGED: the view may be of pages)
template <bool PAGED>
__device__ __forceinline__ KvSeq kv_sequence(const KvView &v, int b) {
  KvSeq s;
  if (v.rd) {
    const RowDesc d = v.rd[(size_t)b * v.rows];
    s.k0 = reinterpret_cast<char *>(global_ptr(reinterpret_cast<char *>(d.k)));
    s.max_pos = d.max_pos;
    s.len = d.pos;
    s.count = d.pos < 0 ? 0 : v.rows;
  } else {
    const bool pages = PAGED && v.table;
    s.k0 = v.base + (pages ? 0 : b * v.seq_bytes);
    s.max_pos = pages ? kv_room(v, b) : v.max_pos;
    s.len = v.lens[b];
    s.count = v.rows;
  }
  if (v.counts) s.count = min(max(v.counts[b], 0), s.count);
  return s;
}
// a byte of the int8 format: the value + 128
__device__ __forceinline__ float kv_byte(uint8_t b) { return (float)((int)b - 128); }
// element e of a word of eight in 4 bits (each the value + 8) times its group's step
__device__ __forceinline__ float kv_nibble(uint32_t word, int e, int step) {
  return (float)(((int)(word >> (4 * e) & 15u) - 8) * step);
}
// The allocation that position p of a sequence is in (its own, or p's page), as a sequence,
// and p's place there: max_pos is the distance of its heads then.
__device__ __forceinline__ KvSeq kv_place(const KvView &v, const KvSeq &s, int b, int &p) {
  if (!v.table) return s;
  KvSeq at = s;
  at.k0 = v.base + kv_page(v, b, p >> v.page_log2) * v.seq_bytes;
  at.max_pos = 1 << v.page_log2;
  p &= at.max_pos - 1;
  return at;
}
// the row of (part: 0 keys, 1 values; kv head g; position p) in rows of the
// sequence's allocation: elements at row * (bytes of a row), scales behind all
// elements, a f32 a row, the 4-bit format's steps behind all scales, a word a row
__device__ __forceinline__ int64_t kv_row(const KvView &v, const KvSeq &s, int part, int g, int p) {
  return (((int64_t)part * v.layers + v.layer) * v.kvh + g) * s.max_pos + p;
}
__device__ __forceinline__ float *kv_scales(const KvView &v, const KvSeq &s, int row_bytes) {
  return reinterpret_cast<float *>(s.k0 + 2 * (int64_t)v.layers * v.kvh * s.max_pos * row_bytes);
}
__device__ __forceinline__ uint32_t *kv_steps(const KvView &v, const KvSeq &s, int row_bytes) {
  return reinterpret_cast<uint32_t *>(kv_scales(v, s, row_bytes) +
                                      2 * (int64_t)v.layers * v.kvh * s.max_pos);
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

// the first sequences of a cache, a layer of it
KvView kv_view(const ::q3h_cache *c, int layer, int sequences, int rows, const int32_t *lens,
               const int32_t *counts);
// what q3h_cache_create refuses of a configuration
void check_cache_config(const ::q3h_cache_config &f, const char *who);

constexpr int kMaxAxes = 4;
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
  // positions of the rows [axis][sequences * rows], the axis of each rotated pair in two
  // bits, and the positions that the table has (places nullable: by length and depth)
  const int32_t *places;
  uint64_t axes[2];
  int n_axes, table_positions;
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
// positions [0, len) of an int8 or 4-bit cache of one sequence (k0: its keys, values
// behind them) from or to f32 [layers][kvh][len][hd]
void launch_scaled_fill(const float *src, char *k0, bool values, int layers, int kvh, int len,
                        int hd, int fmt, int max_pos, hipStream_t st);
void launch_scaled_read(const char *k0, bool values, int layers, int layer, int kvh, int len,
                        int hd, int fmt, int max_pos, float *dst, hipStream_t st);

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
  int axes = 1;                  // axes of positions
  uint64_t pair_axes[2] = {};  // two bits a pair
};

struct q3h_cache {
  q3h_device *dev = nullptr;
  q3h_cache_config cfg{};
  char *data = nullptr;
  size_t seq_bytes = 0;  // of a sequence, or a page
  int64_t bytes = 0;
  // pages (0: none, a sequence's cache in one piece) of 1 << page_log2 positions, up to
  // `slots` a sequence; the table and what its changes need, in one allocation
  int pages = 0, page_log2 = 0, slots = 0;
  int32_t *state = nullptr;
};
