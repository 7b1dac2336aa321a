// q3h_tree.hip - attention of drafted rows over a K/V cache: each row sees the
// positions before the draft and its own path among the drafted rows.
//
// One pass over the cache with the running maximum and sum of a softmax, on
// the matrix cores, without a trip through LDS. The query rows of a kv head
// (drafted row x query head of the group) go in tiles of 16, the positions in
// tiles of 32 (f32: 16):
//   S^T = K Q^T: keys are the rows of the product, queries its columns, so a
//     lane gets scores of one query (lane % 16) for 4 keys of each 16;
//   O^T = V^T P^T: the same lane holds exactly those scores' weights as a
//     column of P^T, where the order of positions along the product's inner
//     dimension is free: V is read in the order the scores have. V^T's rows are
//     the head's elements, dealt so that a lane reads HD / 16 neighbouring ones
//     of a position (whole rows per load instruction) and is left with HD / 4
//     neighbouring elements of its query's output.
// Precision is that of f32 products in every format: f16 and int8 elements are
// exact in f16, queries and weights go in as two f16 parts (22 bits; queries
// scaled to 2^13 .. 2^14 by a power of two per row, weights to at most 2^14, so
// that the second part stays normal), f32 caches use the f32 matrix
// instructions. An int8 row's scale is a factor of the position: it multiplies
// the score, and the weight that the values are summed with. (One f16 part of
// each would be half the products; the sums were then 2^-12 off instead of 2^-21.)
//
// What bounds it, by how much a share has to do (heads of 128):
// - one row over 171 positions of an f16 cache, 8 workgroups of 2 tiles a wave:
//   6.8 us, a launch and the round trips of one workgroup (lengths, rows, the waves'
//   meeting); f32: k_attend_few;
// - 32 sequences of one row, 41000 positions of int8 in all, 87 MB: 25-26 us + 4.8
//   for the parts, 432 shares of 8 steps, where a workgroup takes 10 us to find its
//   share, have its first tiles and join its waves, and 1.45 a step; the same in f16
//   168 MB 44 us, in f32 335 MB 77.6 us (4.3 TB/s). Three workgroups a CU at 168
//   registers (27 us of 23.5), two tiles ahead (29.8 us of 29.1) and loads past the
//   caches (31.2 of 29.3) were slower;
// - a tree of 27 rows over 12289 positions of f16, 51 MB: 22 us + 5.2, 224 shares of 7;
// - 12 trees, 420 rows, 32 query heads over 8, 60000 positions of int8, 141 MB: 130-136
//   us + 11.4 by the box, where VALU (300 instructions a wave and tile, 16 scores a lane taking 9
//   each) and matrix instructions (64) take turns more than they overlap: 69 % and
//   34 % of the time. 260 TFLOP/s of the definition's operations, twice that in
//   products;
// - 2 prompts of 1500 rows over 500 positions, 16 heads over 8: f16 102 us, int8 114,
//   f32 235 (131 of the 154 TFLOP/s of a large f32 product).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "q3h_draft.h"
#include "q3h_wave.h"

namespace q3h {

namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

template <typename T>
__device__ __forceinline__ T load(const char *p, int64_t off) {
  return *reinterpret_cast<const __attribute__((address_space(1))) T *>(
      reinterpret_cast<uintptr_t>(p) + off);
}

// positions of a tile
template <int FMT>
constexpr int kTile = FMT == Q3H_KV_F32 ? 16 : 32;

constexpr float kLog2e = 1.44269504088896340736f;

// How a call is laid out. The query rows of a (sequence, kv head) go in groups of
// `group`, 16 * nq a wave; the waves that a group does not need side by side (wq)
// go over its positions together (wk of them, a tile each: a step). A group's
// steps are cut into shares of about the same length in all groups, a
// workgroup each, so that long and short sequences, full and small groups end
// together; the shares of a group that has several leave parts, which a second
// kernel joins. shares: of a short call no group is cut; blocks: workgroups, of
// shares those that they may come to; parts: that they may leave; workers: how many
// shares of much work there are, about: kWorkers, fewer where the parts of so many
// have no room.
struct Shape {
  int nq, group, blocks, parts;
  bool shares;
  int per_kv;       // query heads of a kv head
  uint32_t by_kv;   // ceil(2^32 / per_kv)
  int workers;
  // x / per_kv (attend_fits: x * per_kv < 2^32)
  __device__ __forceinline__ int drafted(int x) const {
    return per_kv == 1 ? x : (int)__umulhi((uint32_t)x, by_kv);
  }
};

struct Cut {
  int here;    // rows of the group
  int wq, wk;
  int full;    // positions that all its rows see
  int end;     // positions that some row of it sees
  int tiles, steps;
};
__device__ __forceinline__ Cut cut_of(const AttendRows &a, const KvSeq &s, const Shape &shape,
                                      int first, int rows_in, int tile) {
  Cut c;
  c.here = std::min(shape.group, rows_in - first);
  const int turn = c.here > 32 * shape.nq ? 2 : c.here > 16 * shape.nq ? 1 : 0;
  c.wq = 1 << turn;
  c.wk = kWaves >> turn;
  c.full = s.len + (a.parents ? 0 : shape.drafted(first) + 1);
  c.end = s.len + shape.drafted(first + c.here - 1) + 1;
  c.tiles = (c.end + tile - 1) / tile;
  c.steps = (c.tiles + c.wk - 1) >> (2 - turn);
  return c;
}
__device__ __forceinline__ bool bad_length(const AttendRows &a, const KvSeq &s) {
  return s.len < 0 || s.len > a.max_len || s.len > s.max_pos - s.count;
}
// steps of group `first` (of a sequence of a bad length: one, which writes NaN)
__device__ __forceinline__ int group_steps(const AttendRows &a, const KvSeq &s, const Shape &shape,
                                           int first, int rows_in, int tile) {
  return bad_length(a, s) ? 1 : cut_of(a, s, shape, first, rows_in, tile).steps;
}
// a sequence's groups of one kv head: how many, their steps, their shares of up to
// `most` steps, and those of them that leave parts
struct Head {
  int groups, steps, shares, parts;
};
__device__ __forceinline__ Head head_of(const AttendRows &a, const KvSeq &s, const Shape &shape,
                                        int tile, int most) {
  const int rows_in = s.count * shape.per_kv;
  Head h{0, 0, 0, 0};
  for (int first = 0; first < rows_in; first += shape.group) {
    const int n = group_steps(a, s, shape, first, rows_in, tile);
    h.groups++;
    h.steps += n;
    const int k = (n + most - 1) / most;
    h.shares += k;
    h.parts += k > 1 ? k : 0;
  }
  return h;
}
// The steps of a share at most, from all heads' groups and steps. Rounding up
// costs half a share a group: the shares come to about two for each CU, what it
// holds, and to no more than shape.blocks. Of little work one for each CU, as the
// join has twice the parts otherwise and some of the CUs a second share: one row
// over 8000 positions of 8 heads 15.4 us, with two 17.3; a tree of 27 over 12289
// (1544 steps) 26.5 and 29.8; but four rows, 20000 positions in all (1250 steps, 32
// groups) 20.0 and 18.6, four trees 33 and 29.4. (The bound at 16 groups lies between
// what was measured; nothing sets it closer.)
constexpr int kWholeSteps = 6, kWorkers = 512;
__device__ __forceinline__ int share_steps(uint32_t groups, uint32_t steps, uint32_t workers) {
  const uint32_t w = steps <= workers / 2 * (groups < 16 ? 7 : 4) ? workers / 2 : workers;
  const uint32_t n = std::max(w - std::min(groups / 2, w / 2), w / 2);
  return (int)std::max(1u, (steps + n - 1) / n);
}
__device__ __forceinline__ KvSeq lane_sequence(const KvSeq &x, int l) {
  KvSeq s;
  const uint64_t p = reinterpret_cast<uint64_t>(x.k0);
  s.k0 = reinterpret_cast<char *>(
      global_ptr(reinterpret_cast<char *>((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(p >> 32), l) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)p, l))));
  s.max_pos = __builtin_amdgcn_readlane(x.max_pos, l);
  s.len = __builtin_amdgcn_readlane(x.len, l);
  s.count = __builtin_amdgcn_readlane(x.count, l);
  return s;
}

// The workspace of a call: for each part [group][HD] outputs and [group] (maximum,
// sum); the parts before each sequence, and of one of its heads; the steps of a
// share. (A group of k > 1 shares has more than half of k times a share's steps, so
// parts are less than twice the shares that all steps come to.)
struct Parts {
  float *out;
  float2 *ml;
  int32_t *before, *head, *most;  // [sequences], [sequences], [1]
};
inline size_t parts_bytes(const Shape &s, int sequences, int hd) {
  if (!s.shares) return 0;
  return sizeof(float) * s.parts * s.group * (hd + 2) + sizeof(int32_t) * (2 * (size_t)sequences + 1);
}
__device__ __forceinline__ Parts parts_of(const AttendRows &a, const Shape &s, int hd) {
  Parts p;
  const size_t rows = (size_t)s.parts * s.group;
  p.out = a.part;
  p.ml = reinterpret_cast<float2 *>(a.part + rows * hd);
  p.before = reinterpret_cast<int32_t *>(p.ml + rows);
  p.head = p.before + a.kv.sequences;
  p.most = p.head + a.kv.sequences;
  return p;
}
// inclusive sums over the lanes
__device__ __forceinline__ int lane_sums(int x) { return wave_prefix_sum_i(x); }

// two floats rounded to f16 and what is left of them
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
  const h2 h = __builtin_convertvector((f2){x, y}, h2);
  const h2 l = __builtin_convertvector((f2){x - (float)h[0], y - (float)h[1]}, h2);
  hi = __builtin_bit_cast(uint32_t, h);
  lo = __builtin_bit_cast(uint32_t, l);
}

// Two bytes (sel: each under a byte of zeros) of an int8 cache as f16, 2^-9 times
// what they hold, exactly: as subnormals they are 2^-24 times it + 128. (Taken as
// subnormals, sign and magnitude, the matrix instructions lose what is below
// 2^-24 of a normal number: 2^-14 of the smallest byte a product.)
__device__ __forceinline__ uint32_t bytes_f16(uint32_t y, uint32_t x, uint32_t sel) {
  const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(y, x, sel));
  const h2 up = {(_Float16)32768.f, (_Float16)32768.f}, off = {(_Float16)-0.25f, (_Float16)-0.25f};
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(b, up, off));
}

template <int FMT, int HD>
struct Raw;  // a tile's keys and values as loaded

template <int HD>
struct Raw<Q3H_KV_F16, HD> {
  u4 k[2][HD / 32];
  u4 v[8 * HD / 128];  // 8 positions of HD / 16 halves
};
template <int HD>
struct Raw<Q3H_KV_Q8, HD> {
  u4 k[2][HD / 64];
  u2 v[8 * HD / 128];  // 8 positions of HD / 16 bytes
  f4 ks[2], vs[2];
};
template <int HD>
struct Raw<Q3H_KV_F32, HD> {
  f4 k[HD / 16];
  f4 v[4][HD / 64];
};

// NQ query tiles a wave share its loads and conversions of K and V.
template <int FMT, int HD, int NQ>
__global__ __launch_bounds__(kThreads, 2) void k_attend(AttendRows a, Shape shape) {
  constexpr int T = kTile<FMT>;
  constexpr int C = HD / 16;           // output tiles; neighbouring elements a lane reads
  constexpr bool F32 = FMT == Q3H_KV_F32, Q8 = FMT == Q3H_KV_Q8;
  constexpr int NS = F32 ? 1 : 2;                // key tiles of 16 in a tile
  constexpr int ROW = HD * (F32 ? 4 : Q8 ? 1 : 2);  // bytes
  constexpr int LD = HD + 4;  // (rows 4 banks apart)
  // the waves' outputs; before that, with two query tiles a wave, its queries as
  // operands (64 registers: two waves a SIMD would not have them)
  constexpr bool QLDS = NQ > 1 && !F32;
  constexpr int QW = NQ * (HD / 32) * 2 * 256;  // words of a wave's queries
  // with four waves side by side also a tile's keys and values as operands, each
  // wave's quarter
  constexpr int ACC = kWaves * NQ * 16 * LD * 4, QB = QLDS ? kWaves * QW * 4 : 0,
                KVB = QLDS ? T * HD * 2 * 2 : 0, MLB = kWaves * NQ * 16 * 8,
                ML_AT = ACC > QB + KVB - MLB ? ACC : QB + KVB - MLB;  // (not beside a tile)
  __shared__ __align__(16) char sm[ML_AT + MLB];
  float *const sm_acc = reinterpret_cast<float *>(sm);
  float2(*const sm_ml)[NQ * 16] = reinterpret_cast<float2(*)[NQ * 16]>(sm + ML_AT);
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int per_kv = shape.per_kv;
  const int lane = tid & 63;
  // the workgroup's share: steps step0 .. step1 - 1 of group `first` of kv head g
  // of sequence b; whole: all of the group's, else they leave part `slot`
  int b, g, first, step0 = 0, step1 = 0, slot = 0;
  KvSeq s;
  bool whole = true;
  const int n = a.kv.sequences;
  if (!shape.shares) {
    g = blockIdx.x % a.kv.kvh;
    const int bg = blockIdx.x / a.kv.kvh;
    b = bg % n;
    first = bg / n * shape.group;
    s = kv_sequence(a.kv, b);
  } else {
    // each wave finds it by itself, 64 sequences at a time
    KvSeq mine;
    auto head_at = [&](int i, int most) {
      if (most == 1 || n > 64) mine = kv_sequence(a.kv, std::min(i, n - 1));
      return i < n ? head_of(a, mine, shape, T, most) : Head{0, 0, 0, 0};
    };
    Head h{0, 0, 0, 0};
    int groups = 0, steps = 0;
    for (int base = 0; base < n; base += 64) {
      h = head_at(base + lane, 1);
      groups += __builtin_amdgcn_readlane(lane_sums(h.groups), 63) * a.kv.kvh;
      steps += __builtin_amdgcn_readlane(lane_sums(h.steps), 63) * a.kv.kvh;
    }
    const int most = share_steps(groups, steps, shape.workers), worker = blockIdx.x;
    int sum = 0, sum_parts = 0, at = 0, shares = 1, head_parts = 0;
    b = -1;
    for (int base = 0; base < n && (b < 0 || worker == 0); base += 64) {
      h = head_at(base + lane, most);
      const int upto = sum + lane_sums(h.shares) * a.kv.kvh, before = upto - h.shares * a.kv.kvh;
      const int parts_upto = sum_parts + lane_sums(h.parts) * a.kv.kvh,
                parts_before = parts_upto - h.parts * a.kv.kvh;
      if (worker == 0 && tid < 64 && base + lane < n) {
        const Parts p = parts_of(a, shape, HD);
        p.before[base + lane] = parts_before;
        p.head[base + lane] = h.parts;
        *p.most = most;
      }
      const uint64_t hit = __ballot(upto > worker);
      if (b < 0 && hit) {
        const int f = __builtin_ctzll(hit);
        b = base + f;
        at = worker - __builtin_amdgcn_readlane(before, f);
        shares = __builtin_amdgcn_readlane(h.shares, f);
        slot = __builtin_amdgcn_readlane(parts_before, f);
        head_parts = __builtin_amdgcn_readlane(h.parts, f);
        s = lane_sequence(mine, f);
      }
      sum = __builtin_amdgcn_readlane(upto, 63);
      sum_parts = __builtin_amdgcn_readlane(parts_upto, 63);
    }
    // (no share is left; lengths that change while the kernel runs lead nowhere else)
    if (b < 0) return;
    g = at / shares;
    at -= g * shares;
    slot += g * head_parts;
    const int rows_in = s.count * per_kv;
    for (first = 0; first < rows_in; first += shape.group) {
      const int own = group_steps(a, s, shape, first, rows_in, T), k = (own + most - 1) / most;
      if (at < k) {
        // k shares that differ by a step at most
        const int q = own / k, longer = own - q * k;
        step0 = at * q + std::min(at, longer);
        step1 = step0 + q + (at < longer);
        whole = k == 1;
        slot += at;
        break;
      }
      at -= k;
      slot += k > 1 ? k : 0;
    }
  }
  // (as for no share: lengths that change meanwhile)
  if (first >= s.count * per_kv || (!whole && slot >= shape.parts)) return;
  const int n16 = lane & 15, g4 = lane >> 4;
  const int rows_in = s.count * per_kv;  // query rows of the sequence's kv head
  const size_t row0 = (size_t)b * a.kv.rows;
  if (bad_length(a, s)) {
    for (int i = tid; i < shape.group * HD; i += kThreads) {
      const int r = first + i / HD;
      if (r < rows_in)
        a.out[(row0 + r / per_kv) * a.ld_out + (size_t)(g * per_kv + r % per_kv) * HD + i % HD] =
            NAN;
    }
    return;
  }
  const Cut cut = cut_of(a, s, shape, first, rows_in, T);
  const int tile0 = step0 * cut.wk, tile1 = whole ? cut.tiles : std::min(cut.tiles, step1 * cut.wk);
  const int last = cut.end - 1;  // no row behind it is read
  const int here = cut.here, WQ = cut.wq, WK = cut.wk;
  const int wq = wave & (WQ - 1), wk = wave / WQ;

  const char *kbase = s.k0 + kv_row(a.kv, s, 0, g, 0) * ROW;
  const char *vbase = s.k0 + kv_row(a.kv, s, 1, g, 0) * ROW;
  const char *ksc = nullptr, *vsc = nullptr;
  if constexpr (Q8) {
    ksc = reinterpret_cast<const char *>(kv_scales(a.kv, s, HD) + kv_row(a.kv, s, 0, g, 0));
    vsc = reinterpret_cast<const char *>(kv_scales(a.kv, s, HD) + kv_row(a.kv, s, 1, g, 0));
  }

  auto load_scales = [&](const char *sc, int j0, f4(&d)[2]) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
      const int j = j0 + 16 * t + 4 * g4;
      if (j0 + T <= cut.end) {
        d[t] = load<f4u>(sc + 4 * (int64_t)j0, (uint32_t)(64 * t + 16 * g4));
      } else {
#pragma unroll
        for (int r = 0; r < 4; r++) d[t][r] = load<float>(sc, 4 * (int64_t)std::min(j + r, last));
      }
    }
  };
  auto load_k = [&](Raw<FMT, HD> &raw, int tile) {
    const int j0 = tile * T;
    const char *p = kbase + (int64_t)j0 * ROW;
#pragma unroll
    for (int t = 0; t < NS; t++) {
      const uint32_t at = (uint32_t)(std::min(16 * t + n16, last - j0) * ROW + 16 * g4);
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < HD / 16; i++) raw.k[i] = load<f4>(p, at + 64 * i);
      } else if constexpr (Q8) {
#pragma unroll
        for (int i = 0; i < HD / 64; i++) raw.k[t][i] = load<u4>(p, at + 64 * i);
      } else {
#pragma unroll
        for (int i = 0; i < HD / 32; i++) raw.k[t][i] = load<u4>(p, at + 64 * i);
      }
    }
    if constexpr (Q8) load_scales(ksc, j0, raw.ks);
  };
  auto load_v = [&](Raw<FMT, HD> &raw, int tile) {
    const int j0 = tile * T;
    const char *p = vbase + (int64_t)j0 * ROW;
#pragma unroll
    for (int i = 0; i < (F32 ? 4 : 8); i++) {
      const int j = F32 ? 4 * g4 + i : (i >> 2) * 16 + 4 * g4 + (i & 3);
      const uint32_t at = (uint32_t)(std::min(j, last - j0) * ROW + n16 * (ROW / 16));
      if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < HD / 64; e++) raw.v[i][e] = load<f4>(p, at + 16 * e);
      } else if constexpr (Q8) {
        if constexpr (HD == 128) raw.v[i] = load<u2>(p, at);
        else raw.v[i / 2][i & 1] = load<uint32_t>(p, at);
      } else {
        if constexpr (HD == 128) {
          raw.v[i] = load<u4>(p, at);
        } else {
          const u2 x = load<u2>(p, at);
          raw.v[i / 2][2 * (i & 1)] = x[0];
          raw.v[i / 2][2 * (i & 1) + 1] = x[1];
        }
      }
    }
    if constexpr (Q8) load_scales(vsc, j0, raw.vs);
  };
  // word w of the HD / 16 elements of position i of the loaded values
  auto vword = [](const Raw<FMT, HD> &raw, int i, int w) -> uint32_t {
    if constexpr (FMT == Q3H_KV_F16)
      return HD == 128 ? raw.v[i][w] : raw.v[i / 2][2 * (i & 1) + w];
    else if constexpr (Q8)
      return HD == 128 ? raw.v[i][w] : raw.v[i / 2][i & 1];
    else
      return 0;
  };

  // Four waves side by side (more than 64 rows): each loads and converts a quarter
  // of a tile's operands, all take them from LDS (12 trees of up to 64 rows x 4
  // heads, int8: 149 -> 143.6 us; 2 x 1500 rows of a prompt, f16: 105 -> 101.4).
  constexpr int KI = HD / 32, KN = QLDS ? 2 * KI / kWaves : 1, VN = QLDS ? C / kWaves : 1;
  const bool shared = QLDS && WK == 1;
  u4 *const sm_k = reinterpret_cast<u4 *>(sm + QB) + lane, *const sm_v = sm_k + 2 * KI * 64;
  struct Quarter {
    u4 k[Q8 ? 1 : KN];
    uint32_t v[8];
    f4 ks[2], vs[2];
  };
  auto load_quarter = [&](Quarter &raw, int tile) {
    const int j0 = tile * T;
    const int t = wave >> 1, i = (wave & 1) * KN;
    const char *p = kbase + (int64_t)j0 * ROW;
    const uint32_t at = (uint32_t)(std::min(16 * t + n16, last - j0) * ROW + 16 * g4);
    if constexpr (Q8) {
      if constexpr (KN == 2) {
        raw.k[0] = load<u4>(p, at + 32 * i);
      } else {
        const u2 x = load<u2>(p, at + 8 * i);
        raw.k[0][0] = x[0];
        raw.k[0][1] = x[1];
      }
    } else {
#pragma unroll
      for (int u = 0; u < KN; u++) raw.k[u] = load<u4>(p, at + 64 * (i + u));
    }
    p = vbase + (int64_t)j0 * ROW;
    const int word = VN * wave >> (Q8 ? 2 : 1);
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const int j = (u >> 2) * 16 + 4 * g4 + (u & 3);
      raw.v[u] = load<uint32_t>(
          p, (uint32_t)(std::min(j, last - j0) * ROW + n16 * (ROW / 16) + 4 * word));
    }
    if constexpr (Q8) {
      load_scales(ksc, j0, raw.ks);
      load_scales(vsc, j0, raw.vs);
    }
  };
  auto store_quarter = [&](const Quarter &raw) {
#pragma unroll
    for (int u = 0; u < KN; u++) {
      u4 x;
      if constexpr (Q8) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint32_t w = raw.k[0][2 * u + e];
          x[2 * e] = bytes_f16(w, w, 0x0c010c00u);
          x[2 * e + 1] = bytes_f16(w, w, 0x0c030c02u);
        }
      } else {
        x = raw.k[u];
      }
      sm_k[(wave * KN + u) * 64] = x;
    }
#pragma unroll
    for (int u = 0; u < VN; u++) {
      const int c = VN * wave + u;
      // (byte or half c of the words)
      const uint32_t sel = Q8 ? 0x0c040c00u + 0x00010001u * (uint32_t)(c & 3)
                              : c & 1 ? 0x07060302u : 0x05040100u;
      u4 x;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if constexpr (Q8) x[e] = bytes_f16(raw.v[2 * e + 1], raw.v[2 * e], sel);
        else x[e] = __builtin_amdgcn_perm(raw.v[2 * e + 1], raw.v[2 * e], sel);
      }
      sm_v[c * 64] = x;
    }
  };
  auto barrier = [&] {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };

  // the wave's queries: dims of (step, lane group) as the keys' loads have them
  int qrow[NQ], qt[NQ];  // the lane's query row, and the drafted row that it is of
  bool live[NQ];
  f4 qf[F32 ? NQ : 1][HD / 16];
  u4 qh[F32 || QLDS ? 1 : NQ][HD / 32], ql[F32 || QLDS ? 1 : NQ][HD / 32];
  u4 *const qs = reinterpret_cast<u4 *>(sm_acc) + wave * (QW / 4) + lane;
  // the two parts of step i of query tile q
  auto query = [&](int q, int i, int part) -> h8 {
    if constexpr (QLDS) return __builtin_bit_cast(h8, qs[((q * (HD / 32) + i) * 2 + part) * 64]);
    else return __builtin_bit_cast(h8, part ? ql[q][i] : qh[q][i]);
  };
  // a score in powers of two: product (* the key's scale) * sfac, which is above 0
  // (the queries have the scale's sign): the maximum is the products'
  float sfac[NQ];
  const float sign = a.scale < 0.f ? -1.f : 1.f, factor = fabsf(a.scale) * kLog2e;
  f4 qx[NQ][HD / 16];  // as loaded, before the keys and values are on their way
#pragma unroll
  for (int q = 0; q < NQ; q++) {
    const int r = first + (wq * NQ + q) * 16 + n16;
    live[q] = r < rows_in;
    qrow[q] = std::min(r, rows_in - 1);
    qt[q] = shape.drafted(qrow[q]);
    const char *p = reinterpret_cast<const char *>(
        a.q + (row0 + qt[q]) * a.ldq + (size_t)(g * per_kv + qrow[q] - qt[q] * per_kv) * HD);
#pragma unroll
    for (int i = 0; i < HD / 16; i++) {
      const int d = F32 ? 16 * i + 4 * g4
                    : Q8 ? (i >> 2) * 64 + g4 * 16 + (i & 3) * 4
                         : (i >> 1) * 32 + g4 * 8 + (i & 1) * 4;
      qx[q][i] = load<f4u>(p, 4 * d);
    }
  }
  Raw<FMT, HD> raw;
  Quarter quarter;
  int tile = tile0 + wk;
  if (tile < tile1) {
    if (shared) {
      load_quarter(quarter, tile);
    } else {
      load_k(raw, tile);
      load_v(raw, tile);
    }
  }

#pragma unroll
  for (int q = 0; q < NQ; q++) {
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < HD / 16; i++) qf[q][i] = qx[q][i] * sign;
      sfac[q] = factor;
    } else {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 16; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) m = fmaxf(m, fabsf(qx[q][i][e]));
      m = rows4_max(m);
      // m * 2^k in [2^13, 2^14) (rows below 2^-113: less); infinities and NaN stay
      // what they are
      const int k = m > 0.f && m < INFINITY ? std::min(126, 140 - (int)(__float_as_uint(m) >> 23)) : 0;
      const float up = sign * __uint_as_float((uint32_t)(127 + k) << 23);
#pragma unroll
      for (int i = 0; i < HD / 32; i++) {
        u4 h, l;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const f4 x = qx[q][2 * i + (e >> 1)];
          uint32_t hi, lo;
          split2(x[2 * (e & 1)] * up, x[2 * (e & 1) + 1] * up, hi, lo);
          h[e] = hi;
          l[e] = lo;
        }
        if constexpr (QLDS) {
          qs[(q * (HD / 32) + i) * 2 * 64] = h;
          qs[((q * (HD / 32) + i) * 2 + 1) * 64] = l;
        } else {
          qh[q][i] = h;
          ql[q][i] = l;
        }
      }
      sfac[q] = ldexpf(factor, Q8 ? 9 - k : -k);
    }
  }

  f4 acc[NQ][C];
  // The running maximum, and the sum: weights are 2^(score - m). It is less than
  // the scores' maximum by 14 where weights go in as f16, and by 14 - ev of
  // int8 values whose scales are below 2^ev, which are multiplied into the weights:
  // a maximum of scores + ev, so that what goes in is at most 2^14.
  float m[NQ], l[NQ], vmax[NQ];
  uint64_t path[NQ];
  bool broken[NQ], paths = false;
#pragma unroll
  for (int q = 0; q < NQ; q++) {
    path[q] = 0;
    broken[q] = false;
    m[q] = -INFINITY;
    l[q] = vmax[q] = 0.f;
#pragma unroll
    for (int c = 0; c < C; c++) acc[q][c] = (f4){0.f, 0.f, 0.f, 0.f};
  }
  // whether query tile q's row sees drafted row d (d < 0: a position before the draft)
  auto sees = [&](int q, int d) {
    return d < 0 || (d <= qt[q] && (!a.parents || (path[q] >> d & 1)));
  };
  auto step = [&](auto &raw, int tile, auto share) {
    constexpr bool SHARE = decltype(share)::value;
    const int j0 = tile * T, next = tile + WK;
    // (the queries stay in LDS: not read once for all tiles)
    if constexpr (QLDS) asm volatile("" ::: "memory");
    const bool tail = j0 + T > cut.full;
    // scores
    f4 st[NQ][NS];
#pragma unroll
    for (int q = 0; q < NQ; q++)
#pragma unroll
      for (int t = 0; t < NS; t++) st[q][t] = (f4){0.f, 0.f, 0.f, 0.f};
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < HD / 16; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
          for (int q = 0; q < NQ; q++)
            st[q][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(raw.k[i][e], qf[q][i][e], st[q][0], 0,
                                                            0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < HD / 32; i++)
#pragma unroll
        for (int t = 0; t < NS; t++) {
          // int8: the wave at its products goes first, so that the two of a SIMD
          // move apart, one's products beside the other's softmax (143.6 -> 140.1
          // us, the prompt in int8 109.6 -> 111.7; f16 trees slower by 0.5 %)
          if (Q8 && i == 0 && t == 0) __builtin_amdgcn_s_setprio(1);
          u4 ka;
          if constexpr (SHARE) {
            ka = sm_k[(t * KI + i) * 64];
          } else if constexpr (Q8) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const uint32_t w = raw.k[t][i >> 1][2 * (i & 1) + e];
              ka[2 * e] = bytes_f16(w, w, 0x0c010c00u);
              ka[2 * e + 1] = bytes_f16(w, w, 0x0c030c02u);
            }
          } else {
            ka = raw.k[t][i];
          }
          const h8 A = __builtin_bit_cast(h8, ka);
#pragma unroll
          for (int q = 0; q < NQ; q++) {
            st[q][t] =
                __builtin_amdgcn_mfma_f32_16x16x32_f16(A, query(q, i, 1), st[q][t], 0, 0, 0);
            st[q][t] =
                __builtin_amdgcn_mfma_f32_16x16x32_f16(A, query(q, i, 0), st[q][t], 0, 0, 0);
          }
        }
    }
    if constexpr (Q8) __builtin_amdgcn_s_setprio(0);
    f4 ks[2], vs[2];
    if constexpr (Q8) {
#pragma unroll
      for (int t = 0; t < 2; t++) {
        ks[t] = raw.ks[t];
        vs[t] = raw.vs[t];
      }
    }
    if constexpr (SHARE) {
      if (next < tile1) load_quarter(raw, next);
    } else {
      if (next < tile1) load_k(raw, next);
    }

    if (tail && a.parents && !paths) {
      paths = true;
      const Path p = tree_path(a.parents + row0, a.kv.rows);
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        path[q] = __shfl(p.rows, qt[q]);
        broken[q] = __shfl((int)p.bad, qt[q]) != 0;
      }
    }
    // int8: the largest scale of the tile, and whether some are so much smaller
    // (2^16; a weight's two parts have 39 bits below 2^14) that the maximum has to be
    // taken of scores and scales together, position by position. A scale's power of
    // two is taken within 2^-40 .. 2^50: further apart, the factor between two tiles'
    // sums would leave f32. Weights of larger scales leave f16 and become NaN, a wave
    // whose scales are all far smaller is known by the largest: both are done again
    // below.
    float w[NQ][4 * NS], top = 0.f;
    bool wide = tail;
    auto power = [](float x) {
      return (float)std::min(50, std::max(-40, (int)(__float_as_uint(x) >> 23) - 126));
    };
    if constexpr (Q8) {
      float low = INFINITY;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        top = fmaxf(top, vs[i >> 2][i & 3]);
        low = fminf(low, vs[i >> 2][i & 3]);
      }
      top = rows4_max(top);
      wide = wide || __any(low < top * 0x1p-16f);
    }
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      float mx = -INFINITY, vx = top;
#pragma unroll
      for (int i = 0; i < 4 * NS; i++)
        w[q][i] = Q8 ? st[q][i >> 2][i & 3] * ks[i >> 2][i & 3] : st[q][i >> 2][i & 3];
      if (tail) {
        asm volatile("");  // (a branch, so that the other tiles have no selects)
        vx = 0.f;
#pragma unroll
        for (int i = 0; i < 4 * NS; i++) {
          const int d = j0 + (i >> 2) * 16 + 4 * g4 + (i & 3) - s.len;
          const bool see = sees(q, d);
          w[q][i] = see ? w[q][i] : -INFINITY;
          // a row whose path is broken: NaN at itself, and so in all of it
          if (broken[q] && d == qt[q]) w[q][i] = NAN;
          if (Q8 && see) vx = fmaxf(vx, vs[i >> 2][i & 3]);
        }
        if constexpr (Q8) vx = rows4_max(vx);
      }
#pragma unroll
      for (int i = 0; i < 4 * NS; i++) mx = fmaxf(mx, w[q][i]);
      float off = F32 ? 0.f : -14.f;
      if (Q8 && wide) {
        asm volatile("");
        mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4 * NS; i++)
          mx = fmaxf(mx, fmaf(w[q][i], sfac[q], power(vs[i >> 2][i & 3])));
        mx = rows4_max(mx) + off;
      } else {
        mx = fmaf(rows4_max(mx), sfac[q], Q8 ? off + power(top) : off);
      }
      if constexpr (Q8) vmax[q] = fmaxf(vmax[q], vx);
      mx = fmaxf(m[q], mx);
      const float base = mx == -INFINITY ? 0.f : mx;
      if (__any(mx > m[q])) {
        const float f = __builtin_amdgcn_exp2f(m[q] - base);
        l[q] *= f;
#pragma unroll
        for (int c = 0; c < C; c++) acc[q][c] *= f;
        m[q] = mx;
      }
#pragma unroll
      for (int i = 0; i < 4 * NS; i++) {
        const float p = __builtin_amdgcn_exp2f(fmaf(w[q][i], sfac[q], -base));
        l[q] += p;
        w[q][i] = Q8 ? p * vs[i >> 2][i & 3] : p;
      }
    }

    if constexpr (F32) {
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
          for (int q = 0; q < NQ; q++)
            acc[q][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(raw.v[r][c >> 2][c & 3], w[q][r],
                                                             acc[q][c], 0, 0, 0);
    } else {
      h8 ph[NQ], pl[NQ];
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        u4 hi4, lo4;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          uint32_t hi, lo;
          split2(w[q][2 * e], w[q][2 * e + 1], hi, lo);
          hi4[e] = hi;
          lo4[e] = lo;
        }
        ph[q] = __builtin_bit_cast(h8, hi4);
        pl[q] = __builtin_bit_cast(h8, lo4);
      }
#pragma unroll
      for (int c = 0; c < C; c++) {
        if (Q8 && c == 0) __builtin_amdgcn_s_setprio(1);
        u4 va;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if constexpr (SHARE) {
            // (below)
          } else if constexpr (Q8) {
            // bytes c of positions 2e and 2e + 1
            va[e] = bytes_f16(vword(raw, 2 * e + 1, c >> 2), vword(raw, 2 * e, c >> 2),
                              0x0c040c00u + 0x00010001u * (c & 3));
          } else {
            const uint32_t x = vword(raw, 2 * e, c >> 1), y = vword(raw, 2 * e + 1, c >> 1);
            va[e] = __builtin_amdgcn_perm(y, x, c & 1 ? 0x07060302u : 0x05040100u);
          }
        }
        if constexpr (SHARE) va = sm_v[c * 64];
        const h8 A = __builtin_bit_cast(h8, va);
#pragma unroll
        for (int q = 0; q < NQ; q++) {
          acc[q][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, pl[q], acc[q][c], 0, 0, 0);
          acc[q][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, ph[q], acc[q][c], 0, 0, 0);
        }
      }
    }
    if constexpr (Q8) __builtin_amdgcn_s_setprio(0);
    if constexpr (!SHARE) {
      if (next < tile1) load_v(raw, next);
    }
  };
  if (shared) {
    if constexpr (QLDS) {
      for (; tile < tile1; tile++) {
        store_quarter(quarter);
        barrier();
        step(quarter, tile, std::true_type());
        barrier();
      }
    }
  } else {
    for (; tile < tile1; tile += WK) step(raw, tile, std::false_type());
  }

  // what the outputs are still to be multiplied with; whether any is NaN (or, as
  // good, infinite)
  float scale[NQ];
  bool nan = false;
#pragma unroll
  for (int q = 0; q < NQ; q++) {
    scale[q] = Q8 ? 0x1p9f : 1.f;
    l[q] = rows4_sum(l[q]);
    float zero = 0.f * l[q];
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int r = 0; r < 4; r++) zero = fmaf(acc[q][c][r], 0.f, zero);
    nan = nan || (zero != 0.f && !broken[q]) || (Q8 && vmax[q] > 0.f && vmax[q] < 0x1p-56f);
  }
  // An infinity times one of the parts that a query or a weight is split in is
  // NaN where the product itself is not, and so is an infinity that a row does
  // not see times its weight 0. A wave that ends with a NaN goes over its
  // positions again one by one, each lane on its query and its HD / 4 elements.
  if (__any(nan)) {
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      const float *p = a.q + (row0 + qt[q]) * a.ldq +
                       (size_t)(g * per_kv + qrow[q] - qt[q] * per_kv) * HD + C * 4 * g4;
      float ms = -INFINITY, ls = 0.f;
#pragma unroll
      for (int c = 0; c < C; c++) acc[q][c] = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int at = tile0 + wk; at < tile1; at += WK)
#pragma unroll 1
        for (int j = at * T; j < std::min(at * T + T, cut.end); j++) {
          const float kd = Q8 ? load<float>(ksc, 4 * (int64_t)j) : 1.f;
          const float vd = Q8 ? load<float>(vsc, 4 * (int64_t)j) : 1.f;
          auto value = [&](const char *base, int e) {
            const int64_t off = (int64_t)j * ROW;
            if constexpr (F32) return load<float>(base, off + 4 * e);
            else if constexpr (Q8) return kv_byte(load<uint8_t>(base, off + e));
            else return (float)load<_Float16>(base, off + 2 * e);
          };
          float x = 0.f;
#pragma unroll 1
          for (int e = 0; e < HD / 4; e++) x = fmaf(p[e], value(kbase, C * 4 * g4 + e), x);
          x = rows4_sum(x) * kd * a.scale * kLog2e;
          if (!sees(q, j - s.len)) continue;
          if (broken[q]) x = NAN;
          const float mn = fmaxf(ms, x), base = mn == -INFINITY ? 0.f : mn;
          const float f = __builtin_amdgcn_exp2f(ms - base), w = __builtin_amdgcn_exp2f(x - base);
          ls = fmaf(ls, f, w);
#pragma unroll
          for (int c = 0; c < C; c++)
#pragma unroll
            for (int r = 0; r < 4; r++)
              acc[q][c][r] = fmaf(acc[q][c][r], f, w * (value(vbase, C * (4 * g4 + r) + c) * vd));
          ms = mn;
        }
      m[q] = ms;
      l[q] = ls;
      scale[q] = 1.f;
    }
  }

  // the waves over the positions together
  constexpr int Q16 = NQ * 16;
  if (WK > 1) {
    if (g4 == 0) {
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        sm_ml[wave][q * 16 + n16] = make_float2(m[q], l[q]);
      }
    }
    __syncthreads();
  }
  const Parts parts = parts_of(a, shape, HD);
  const size_t part0 = (size_t)slot * shape.group - first;
#pragma unroll
  for (int q = 0; q < NQ; q++) {
    float M = m[q], L = l[q], f = 1.f;
    if (WK > 1) {
      // (of two waves each twice: the maximum stays, and a sum counts half)
      float2 o[kWaves];
#pragma unroll
      for (int i = 0; i < kWaves; i++) o[i] = sm_ml[(i * WQ + wq) & (kWaves - 1)][q * 16 + n16];
      M = fmaxf(fmaxf(o[0].x, o[1].x), fmaxf(o[2].x, o[3].x));
      const float base = M == -INFINITY ? 0.f : M;
      L = 0.f;
#pragma unroll
      for (int i = 0; i < kWaves; i++) L += o[i].y * __builtin_amdgcn_exp2f(o[i].x - base);
      if (WK == 2) L *= 0.5f;
      f = __builtin_amdgcn_exp2f(m[q] - base);
    }
    f *= scale[q];
    if (whole) f /= L;  // the softmax's sum
    if (!whole && wk == 0 && g4 == 0 && live[q]) parts.ml[part0 + qrow[q]] = make_float2(M, L);
    if (!live[q]) continue;
    float *o = WK > 1 ? sm_acc + (wave * Q16 + q * 16 + n16) * LD
               : !whole
                   ? parts.out + (part0 + qrow[q]) * HD
                   : a.out + (row0 + qt[q]) * a.ld_out +
                         (size_t)(g * per_kv + qrow[q] - qt[q] * per_kv) * HD;
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int c = 0; c < C; c += 4) {
        const f4 x = {acc[q][c][r] * f, acc[q][c + 1][r] * f, acc[q][c + 2][r] * f,
                      acc[q][c + 3][r] * f};
        if (WK > 1) *reinterpret_cast<f4 *>(o + C * (4 * g4 + r) + c) = x;
        else *reinterpret_cast<f4u *>(o + C * (4 * g4 + r) + c) = x;
      }
  }
  if (WK > 1) {
    __syncthreads();
    for (int i = tid; i < here * (HD / 4); i += kThreads) {
      const int r = i / (HD / 4), e = i % (HD / 4) * 4;  // row of the group
      const int row = first + r;
      f4 x = {0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < WK; k++)
        x += *reinterpret_cast<const f4 *>(
            sm_acc + ((k * WQ + r / Q16) * Q16 + r % Q16) * LD + e);
      float *o = parts.out + (part0 + row) * HD;
      if (whole) {
        const int t = shape.drafted(row);
        o = a.out + (row0 + t) * a.ld_out + (size_t)(g * per_kv + row - t * per_kv) * HD;
      }
      *reinterpret_cast<f4u *>(o + e) = x;
    }
  }
}

// One or two query rows of a kv head over an f32 cache, uncut: the f32 matrix
// instructions would spend 14 of their 16 columns on nothing (2048 cycles a tile of
// 16 positions; here 220 instructions). A wave's tile: a score per lane (position
// lane % 16, summed over four lanes of HD / 4 elements each), then the values with
// HD / 64 elements a lane, their weights broadcast. Bound by its round trips
// (lengths, rows and queries, the waves' meeting): 171 positions, 16 heads over 8,
// 8.1 us (8.9 on the matrix instructions; 8.6 with four waves, 8.2 with eight), 64
// such sequences 14.1 (16.5).
template <int HD>
__global__ __launch_bounds__(384) void k_attend_few(AttendRows a, int per_kv) {
  constexpr int R = 2, W = 6, E = HD / 64;
  typedef float fe __attribute__((ext_vector_type(E)));
  __shared__ fe sm_acc[W][R][64];
  __shared__ float2 sm_ml[W][R];
  auto row_max = [](float v) {  // of the lane's row of 16
    v = quad_max_dpp(v);
    v = fmaxf(v, dpp_f_keep<kHalfMirror>(v));
    return fmaxf(v, dpp_f_keep<kRowMirror>(v));
  };
  auto row_sum = [](float v) {
    v += dpp_f<kQuadXor1>(v);
    v += dpp_f<kQuadXor2>(v);
    v += dpp_f<kHalfMirror>(v);
    return v + dpp_f<kRowMirror>(v);
  };
  const int lane = threadIdx.x & 63, n16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.x / a.kv.kvh, g = blockIdx.x - b * a.kv.kvh;
  const KvSeq s = kv_sequence(a.kv, b);
  const int rows_in = s.count * per_kv;
  if (rows_in < 1) return;
  const size_t row0 = (size_t)b * a.kv.rows;
  // query row r: drafted row r / per_kv (0 or r)
  auto drafted = [&](int r) { return per_kv == 1 ? r : 0; };
  auto out = [&](int r) {
    return a.out + (row0 + drafted(r)) * a.ld_out + (size_t)(g * per_kv + r - drafted(r) * per_kv) * HD;
  };
  if (bad_length(a, s)) {
    for (int i = threadIdx.x; i < rows_in * HD; i += 64 * W) out(i / HD)[i % HD] = NAN;
    return;
  }
  const int end = s.len + s.count, last = end - 1;
  const char *kbase = s.k0 + kv_row(a.kv, s, 0, g, 0) * (HD * 4);
  const char *vbase = s.k0 + kv_row(a.kv, s, 1, g, 0) * (HD * 4);
  f4 q[R][HD / 16];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const int at = std::min(r, rows_in - 1), t = drafted(at);
    const char *p = reinterpret_cast<const char *>(
        a.q + (row0 + t) * a.ldq + (size_t)(g * per_kv + at - t * per_kv) * HD);
#pragma unroll
    for (int i = 0; i < HD / 16; i++) q[r][i] = load<f4u>(p, 4 * (16 * i + 4 * g4));
  }
  // the second of two drafted rows sees the first one if it continues it
  const int parent = a.parents && s.count > 1 ? a.parents[row0 + 1] : 0;
  const int root = a.parents ? a.parents[row0] : -1;
  const float factor = a.scale * kLog2e;
  float m[R] = {-INFINITY, -INFINITY}, l[R] = {0.f, 0.f};
  fe acc[R] = {};
  for (int tile = wave; tile * 16 < end; tile += W) {
    const int j0 = tile * 16;
    const char *kp = kbase + (int64_t)j0 * (HD * 4), *vp = vbase + (int64_t)j0 * (HD * 4);
    f4 k[HD / 16];
    fe v[16];
#pragma unroll
    for (int i = 0; i < HD / 16; i++)
      k[i] = load<f4>(kp, (uint32_t)(std::min(n16, last - j0) * HD * 4 + 64 * i + 16 * g4));
#pragma unroll
    for (int j = 0; j < 16; j++)
      v[j] = load<fe>(vp, (uint32_t)(std::min(j, last - j0) * HD * 4 + 4 * E * lane));
    float w[R];
    uint32_t seen[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 16; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) x = fmaf(k[i][e], q[r][i][e], x);
      x = rows4_sum(x) * factor;
      const int d = j0 + n16 - s.len, t = drafted(r);
      const bool see = d < 0 || d == t || (t == 1 && d == 0 && parent == 0);
      seen[r] = (uint32_t)__ballot(see) & 0xffffu;
      x = see ? x : -INFINITY;
      const float mx = fmaxf(m[r], row_max(x)), base = mx == -INFINITY ? 0.f : mx;
      const float f = __builtin_amdgcn_exp2f(m[r] - base);
      w[r] = __builtin_amdgcn_exp2f(x - base);
      l[r] = fmaf(l[r], f, w[r]);
      acc[r] *= f;
      m[r] = mx;
    }
#pragma unroll
    for (int j = 0; j < 16; j++)
#pragma unroll
      for (int r = 0; r < R; r++)
        if (seen[r] >> j & 1) acc[r] += lane_f(w[r], j) * v[j];
  }
#pragma unroll
  for (int r = 0; r < R; r++) {
    // (each of the four lane groups has all positions)
    l[r] = row_sum(l[r]);
    sm_acc[wave][r][lane] = acc[r];
    if (lane == 0) sm_ml[wave][r] = make_float2(m[r], l[r]);
  }
  __syncthreads();
  if (wave >= rows_in) return;
  const int r = wave;
  float M = -INFINITY, L = 0.f;
#pragma unroll
  for (int i = 0; i < W; i++) M = fmaxf(M, sm_ml[i][r].x);
  const float base = M == -INFINITY ? 0.f : M;
  fe x = {};
#pragma unroll
  for (int i = 0; i < W; i++) {
    const float f = __builtin_amdgcn_exp2f(sm_ml[i][r].x - base);
    L = fmaf(sm_ml[i][r].y, f, L);
    x += sm_acc[i][r][lane] * f;
  }
  // a parent that is not below its row, on the row's path
  const bool bad = root >= 0 || root < -1, bad1 = parent > 0 || parent < -1;
  const int t = drafted(r);
  const bool broken = t == 0 ? bad : bad1 || (parent == 0 && bad);
  typedef float feu __attribute__((ext_vector_type(E), aligned(4)));
  *(reinterpret_cast<feu *>(out(r)) + lane) = broken ? x * NAN : x / L;
}

// The parts of the rows whose group has several shares, joined. A wave takes
// neighbouring rows of a group, HD / 4 lanes each, so that it finds its parts once
// for 256 / HD rows and asks for them in 16 bytes a lane; or four waves do, each
// over every fourth part (side 4).
template <int HD>
__global__ __launch_bounds__(kThreads) void k_attend_join(AttendRows a, Shape shape, int tile,
                                                          int side) {
  constexpr int R = 256 / HD, AHEAD = 4;
  __shared__ f4 sm[kWaves][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per_kv = shape.per_kv;
  const int sets = (a.kv.rows * per_kv + R - 1) / R;
  const int id = side == 1 ? blockIdx.x * kWaves + wave : blockIdx.x;
  const int bg = id / sets, row0 = (id - bg * sets) * R;
  const int b = bg / a.kv.kvh, g = bg - b * a.kv.kvh;
  if (b >= a.kv.sequences) return;
  const KvSeq s = kv_sequence(a.kv, b);
  const Parts parts = parts_of(a, shape, HD);
  const int most = *parts.most;
  int start = parts.before[b] + g * parts.head[b], n = 1;
  const int rows_in = s.count * per_kv;
  if (row0 >= rows_in) return;
  const int mine = row0 / shape.group * shape.group;
  for (int first = 0; first <= mine; first += shape.group) {
    start += n > 1 ? n : 0;
    n = (group_steps(a, s, shape, first, rows_in, tile) + most - 1) / most;
  }
  if (n <= 1 || start < 0 || start + n > shape.parts) return;  // (one share: written as it is)
  const int sub = lane / (HD / 4), e = lane % (HD / 4) * 4;
  auto part = [&](int i, int r) {
    return (size_t)(start + i) * shape.group + (std::min(row0 + r, rows_in - 1) - mine);
  };
  float M[R], L[R];
  float2 head[R];  // of the first 64 parts
#pragma unroll
  for (int r = 0; r < R; r++) {
    head[r] = lane < n ? parts.ml[part(lane, r)] : make_float2(-INFINITY, 0.f);
    M[r] = head[r].x;
    L[r] = 0.f;
  }
  for (int i = lane + 64; i < n; i += 64)
#pragma unroll
    for (int r = 0; r < R; r++) M[r] = fmaxf(M[r], parts.ml[part(i, r)].x);
#pragma unroll
  for (int r = 0; r < R; r++) {
    M[r] = wave_max_dpp(M[r]);
    if (M[r] == -INFINITY) M[r] = 0.f;
  }
  f4 x = {0.f, 0.f, 0.f, 0.f};
  const int step = side == 1 ? 1 : kWaves;
  for (int base = 0; base < n; base += 64) {
    float f[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      float2 p = head[r];
      if (base > 0)
        p = base + lane < n ? parts.ml[part(base + lane, r)] : make_float2(-INFINITY, 0.f);
      f[r] = __builtin_amdgcn_exp2f(p.x - M[r]);
      L[r] += wave_sum_dpp(p.y * f[r]);
    }
    const int end = min(n, base + 64);
    for (int i0 = base + (side == 1 ? 0 : wave); i0 < end; i0 += AHEAD * step) {
      f4 y[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; i++)
        y[i] = *reinterpret_cast<const f4 *>(
            parts.out + part(min(i0 + i * step, end - 1), sub) * HD + e);
#pragma unroll
      for (int i = 0; i < AHEAD; i++)
        if (i0 + i * step < end) {
          float k = lane_f(f[0], i0 + i * step - base);
#pragma unroll
          for (int r = 1; r < R; r++) {
            const float other = lane_f(f[r], i0 + i * step - base);
            k = sub == r ? other : k;
          }
          x += k * y[i];
        }
    }
  }
  if (side > 1) {
    sm[wave][lane] = x;
    __syncthreads();
    if (wave > 0) return;
    x = (sm[0][lane] + sm[1][lane]) + (sm[2][lane] + sm[3][lane]);
  }
  float sum = L[0];
#pragma unroll
  for (int r = 1; r < R; r++) sum = sub == r ? L[r] : sum;
  const int row = row0 + sub;
  if (row >= rows_in) return;
  const int t = shape.drafted(row);
  *reinterpret_cast<f4u *>(a.out + ((size_t)b * a.kv.rows + t) * a.ld_out +
                           (size_t)(g * per_kv + row - t * per_kv) * HD + e) = x / sum;
}

// steps of a call at most (a product that can leave 64 bits)
double steps_upto(int sequences, int rows, int heads, int kvh, int max_len, int tile) {
  return (double)(((int64_t)rows * (heads / kvh) + 15) / 16) * sequences * kvh *
         ((max_len + rows + tile - 1) / tile);
}

// room: bytes that the parts have
Shape shape_of(int sequences, int rows, int heads, int kvh, int hd, int max_len, int tile,
               size_t room) {
  Shape s;
  s.per_kv = heads / kvh;
  s.by_kv = (uint32_t)(((1ull << 32) + s.per_kv - 1) / s.per_kv);
  const int q_rows = rows * s.per_kv;
  s.nq = q_rows > 16 ? 2 : 1;
  const int waves = q_rows > 32 * s.nq ? 4 : q_rows > 16 * s.nq ? 2 : 1;
  s.group = 16 * s.nq * waves;
  const int64_t groups = (int64_t)sequences * kvh * ((q_rows + s.group - 1) / s.group);
  const int wk = kWaves / waves;
  const int64_t steps = ((max_len + rows + tile - 1) / tile + wk - 1) / wk;
  // Up to six steps no group is cut: parts cost a second launch, 4 us (one row over
  // 640 positions of f16: 11.1 us whole, 12.5 cut; 900: 14.4 and 11.9; the other formats
  // take the same number, f32 with half the positions a step). Beyond, the
  // more workgroups the better, down to one step each (8000 positions: 18.5 us with
  // six steps at least, 15.4 with one or two).
  s.shares = steps > kWholeSteps;
  for (int w = s.workers = kWorkers; s.shares && w > 0; w -= kWorkers / 16) {
    const int64_t n = std::max<int64_t>(w - groups / 2, w / 2);
    s.workers = w;
    s.blocks = (int)std::min(n + groups, groups * steps);
    // n shares of whole steps and one more a group, or twice n: the most of any number
    // of groups up to these is at a third of 2 w
    s.parts = (int)std::min<int64_t>(w + std::min<int64_t>(groups, 2 * w / 3) / 2 + 2, s.blocks);
    if (parts_bytes(s, sequences, hd) <= room) return s;
  }
  // short, or no room for the parts of any cut: whole groups
  s.shares = false;
  s.blocks = (int)groups;
  s.parts = 0;
  return s;
}

// sets of rows that k_attend_join has a wave for
int64_t join_sets(int sequences, int rows, int heads, int kvh, int hd) {
  const int64_t per = 256 / hd;
  return (int64_t)sequences * kvh * (((int64_t)rows * (heads / kvh) + per - 1) / per);
}

template <int FMT, int HD>
void launch(const AttendRows &a, hipStream_t st) {
  const Shape s = shape_of(a.kv.sequences, a.kv.rows, a.heads, a.kv.kvh, HD, a.max_len, kTile<FMT>,
                           a.room);
  const unsigned blocks = s.blocks;
  if (FMT == Q3H_KV_F32 && !s.shares && a.kv.rows * s.per_kv <= 2) {
    hipLaunchKernelGGL((k_attend_few<HD>), dim3(blocks), dim3(384), 0, st, a, s.per_kv);
    return;
  }
  if (s.nq == 1)
    hipLaunchKernelGGL((k_attend<FMT, HD, 1>), dim3(blocks), dim3(kThreads), 0, st, a, s);
  else
    hipLaunchKernelGGL((k_attend<FMT, HD, 2>), dim3(blocks), dim3(kThreads), 0, st, a, s);
  if (s.shares) {
    const int64_t sets = join_sets(a.kv.sequences, a.kv.rows, a.heads, a.kv.kvh, HD);
    const int side = sets >= 2048 ? 1 : kWaves;
    hipLaunchKernelGGL((k_attend_join<HD>),
                       dim3((unsigned)(side == 1 ? (sets + kWaves - 1) / kWaves : sets)),
                       dim3(kThreads), 0, st, a, s, kTile<FMT>, side);
  }
}

}  // namespace

size_t attend_part_bytes(int sequences, int rows, int heads, int kvh, int hd, int fmt,
                         int max_len) {
  return parts_bytes(shape_of(sequences, rows, heads, kvh, hd, max_len, fmt == Q3H_KV_F32 ? 16 : 32,
                              SIZE_MAX),
                     sequences, hd);
}

bool attend_fits(int sequences, int rows, int heads, int kvh, int hd, int fmt, int max_len) {
  const int64_t per_kv = heads / kvh, most = (int64_t)1 << 32;  // threads of a launch: below
  const int tile = fmt == Q3H_KV_F32 ? 16 : 32;
  // (steps in 32 bits, and with them groups and shares)
  if (rows * per_kv * per_kv >= most ||
      steps_upto(sequences, rows, heads, kvh, max_len, tile) > 0x1p30)
    return false;
  const Shape s = shape_of(sequences, rows, heads, kvh, hd, max_len, tile, SIZE_MAX);
  return (int64_t)s.blocks * 512 < most &&
         (!s.shares || join_sets(sequences, rows, heads, kvh, hd) * 64 + kThreads < most);
}

void launch_cache_attend(const AttendRows &a, int hd, int fmt, hipStream_t st) {
  if (hd == 64) {
    if (fmt == Q3H_KV_F32) launch<Q3H_KV_F32, 64>(a, st);
    else if (fmt == Q3H_KV_F16) launch<Q3H_KV_F16, 64>(a, st);
    else launch<Q3H_KV_Q8, 64>(a, st);
  } else {
    if (fmt == Q3H_KV_F32) launch<Q3H_KV_F32, 128>(a, st);
    else if (fmt == Q3H_KV_F16) launch<Q3H_KV_F16, 128>(a, st);
    else launch<Q3H_KV_Q8, 128>(a, st);
  }
}

}  // namespace q3h
