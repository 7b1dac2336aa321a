// q3h_cache.hip - a K/V cache of several sequences: rotary tables, the append
// of drafted rows (norm, rotation, rounding to the cache's format), reading
// back, and moving the kept rows to the front.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>
#include <vector>

#include "q3h.h"
#include "q3h_api_internal.h"
#include "q3h_draft.h"
#include "q3h_wave.h"

namespace q3h {

namespace {

constexpr int kThreads = 256;

// table [positions][pairs] of (cos, sin) * mag at position * freq, in 64 bits
__global__ void k_rope_table(const double *freq, double mag, int pairs, size_t n, double2 *table) {
  const size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  double s, c;
  sincos((double)(i / pairs) * freq[i % pairs], &s, &c);
  table[i] = make_double2(c * mag, s * mag);
}

// sum and maximum over the L lanes (8 or 16, a row of lanes or half of one) of a
// head, in every lane
template <int L>
__device__ __forceinline__ double head_sum(double v) {
#pragma unroll
  for (int i = 0; i < (L == 16 ? 4 : 3); i++) v += dpp_d_step(v, i);
  return v;
}
template <int L>
__device__ __forceinline__ float head_max(float v) {
  v = fmaxf(v, dpp_f_keep<kQuadXor1>(v));
  v = fmaxf(v, dpp_f_keep<kQuadXor2>(v));
  v = fmaxf(v, dpp_f_keep<kHalfMirror>(v));
  return L == 16 ? fmaxf(v, dpp_f_keep<kRowMirror>(v)) : v;
}

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

// rint(x / d) for the bytes of a row: the quotient by the reciprocal, by the
// division itself where a reciprocal's error could cross a half
__device__ __forceinline__ int byte_of(float x, float d, double inv) {
  double y = (double)x * inv, q = rint(y);
  if (fabs(y - q) > 0.5 - 1e-6) q = rint((double)x / (double)d);
  return min(127, max(-127, (int)q)) + 128;
}

// One head of one row per HD / 8 lanes, twice four neighbours each, a and b, such
// that a head's lanes together load and store whole lines: a[i] and b[i] of four
// pairs that turn together (halves), four pairs of neighbours (interleaved), or
// elements that do not turn. A wave has 512 / HD heads of a row side by side,
// kHeads of them one after another with one square root and division for all,
// and goes over the row's heads with the same turning angles; loads and stores
// are of 16 bytes a lane (f16: 8, int8: 4). ODD: pairs that are not a multiple of
// four, element by element. Everything up to the f32 row is in 64 bits, so that a
// byte of the int8 format is that of the definition and not of a rounding
// before it: y = x / sqrt(sum x^2 / HD + eps) * w; (y0 c - y1 s, y1 c + y0 s);
// d = fl32(max |y| / 127), byte = rint(y / d).
//
// Memory bound over many rows: 3576 rows of 32 + 2 x 8 heads of 128 to f16, 161 MB
// read and written, 32 us (5.0 TB/s; turning 20 of the 128 elements, ODD, three times
// that; eight neighbours a lane, half of a line an
// instruction, 38; a pair a lane, a head over a whole wave, 60: the 64-bit sums of
// each head made that VALU bound). One row: 3.6 us, 496 rows of 16 + 2 x 8 heads to
// int8 7.4 us, which are a launch, the path through the parents and three loads that
// wait for each other (length, angles, rows).
constexpr int kHeads = 2, kManyRows = 1024;
template <int FMT, int HD, bool ODD, bool MANY>
__global__ __launch_bounds__(kThreads) void k_cache_append(AppendRows a) {
  constexpr int G = HD / 8, SIDE = 64 / G;  // lanes of a head, heads side by side
  constexpr int PER = kHeads * SIDE;        // heads of a wave at a time
  const int lane = threadIdx.x & 63, sub = lane & (G - 1), side = lane / G;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x, b = row / a.kv.rows, t = row - b * a.kv.rows;
  const KvSeq s = kv_sequence(a.kv, b);
  if (t >= s.count) return;
  int depth = t;
  bool bad = s.len < 0 || s.len > s.max_pos - s.count;
  if (a.parents) {
    const Path path = tree_path(a.parents + (size_t)b * a.kv.rows, a.kv.rows);
    depth = __shfl(path.depth, t);
    bad = bad || __shfl((int)path.bad, t) != 0;
  }
  const int kvh = a.kv.kvh, turned = a.heads + kvh;
  const bool rotary = a.table || a.table32;
  const int half = rotary ? a.rot_dim >> 1 : 0;
  // the lane's elements: four from ea, four from eb (ODD: e[i] and e[4 + i])
  const bool split = rotary && !a.interleaved;
  bool turns = 4 * sub < half, turns_b = turns;  // (interleaved: of the first and the last four)
  int ea = 4 * sub, eb = HD / 2 + ea;
  if (split) {
    ea = turns ? 4 * sub : a.rot_dim + 4 * sub - half;
    eb = turns ? half + 4 * sub : ea + (HD - a.rot_dim) / 2;
  } else {
    turns = 2 * sub < half;
    turns_b = HD / 4 + 2 * sub < half;
  }
  int e[ODD ? 8 : 1];
  if constexpr (ODD) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int p = 4 * sub + i;
      e[i] = !split ? 2 * p : p < half ? p : a.rot_dim + 2 * (p - half);
      e[4 + i] = split && p < half ? half + p : e[i] + 1;
    }
  }
  double2 cs[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int p = ODD || split ? 4 * sub + i : (i < 2 ? 2 * sub + i : HD / 4 + 2 * sub + i - 2);
    cs[i] = make_double2(1.0, 0.0);
    if (p < half && !bad) {
      const size_t at = (size_t)(s.len + depth) * half + p;
      if (a.table) {
        cs[i] = a.table[at];
      } else {
        const float2 c = a.table32[at];
        cs[i] = make_double2(c.x, c.y);
      }
    }
  }
  auto load8 = [&](const float *p, float (&x)[8], bool values) {
    if (ODD && !values) {
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = p[e[ODD ? i : 0]];
    } else {
      const f4u w0 = *reinterpret_cast<const f4u *>(p + (values ? 4 * sub : ea));
      const f4u w1 = *reinterpret_cast<const f4u *>(p + (values ? HD / 2 + 4 * sub : eb));
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[i] = w0[i];
        x[4 + i] = w1[i];
      }
    }
  };
  const float *src_q = a.q + (size_t)row * a.ldq, *src_k = a.k + (size_t)row * a.ldk,
              *src_v = a.v + (size_t)row * a.ldv;
  const int groups = (turned + PER - 1) / PER, all = groups + (kvh + PER - 1) / PER;
  for (int group = blockIdx.y * (kThreads / 64) + wave; group < all;
       group += gridDim.y * (kThreads / 64)) {
    const bool values = group >= groups;
    const int first = (values ? group - groups : group) * PER + side;
    const int heads = values ? kvh : turned;
    float x[kHeads][8];
#pragma unroll
    for (int u = 0; u < kHeads; u++) {
      const int j = min(first + u * SIDE, heads - 1);
      load8(values ? src_v + (size_t)j * HD
                   : j < a.heads ? src_q + (size_t)j * HD
                                 : src_k + (size_t)(j - a.heads) * HD,
            x[u], values);
    }
    if (!values) {
      double y[kHeads][8];
#pragma unroll
      for (int u = 0; u < kHeads; u++)
#pragma unroll
        for (int i = 0; i < 8; i++) y[u][i] = x[u][i];
      if (a.q_norm || a.k_norm) {
        double ss[kHeads];
#pragma unroll
        for (int u = 0; u < kHeads; u++) {
          ss[u] = 0.0;
#pragma unroll
          for (int i = 0; i < 8; i++) ss[u] += y[u][i] * y[u][i];
          ss[u] = head_sum<G>(ss[u]);
        }
        // lane u of a head does the u-th one's root
        double mine = ss[0];
#pragma unroll
        for (int u = 1; u < kHeads; u++) mine = sub == u ? ss[u] : mine;
        const double inv = 1.0 / sqrt(mine / HD + (double)a.eps);
#pragma unroll
        for (int u = 0; u < kHeads; u++) {
          const double f = __shfl(inv, side * G + u);
          const float *w = min(first + u * SIDE, heads - 1) < a.heads ? a.q_norm : a.k_norm;
          if (w) {
            float wx[8];
            load8(w, wx, false);
#pragma unroll
            for (int i = 0; i < 8; i++) y[u][i] = y[u][i] * f * (double)wx[i];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kHeads; u++) {
        auto turn = [&](double &y0, double &y1, int i) {
          const double r0 = y0 * cs[i].x - y1 * cs[i].y;
          y1 = y1 * cs[i].x + y0 * cs[i].y;
          y0 = r0;
        };
        if constexpr (ODD) {
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (4 * sub + i < half) turn(y[u][i], y[u][4 + i], i);
        } else if (split) {
          if (turns) {
#pragma unroll
            for (int i = 0; i < 4; i++) turn(y[u][i], y[u][4 + i], i);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (i < 2 ? turns : turns_b) turn(y[u][2 * i], y[u][2 * i + 1], i);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) x[u][i] = (float)y[u][i];
      }
    }
    // the int8 format: the heads' scales
    float d[kHeads] = {};
    double inv[kHeads] = {};
    if constexpr (FMT == Q3H_KV_Q8) {
      if (values || (group + 1) * PER > a.heads) {
        float m[kHeads];
#pragma unroll
        for (int u = 0; u < kHeads; u++) {
          // (fmaxf drops a NaN: it is found by its comparison)
          float most = 0.f;
          bool finite = true;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            finite = finite && fabsf(x[u][i]) < INFINITY;
            most = fmaxf(most, fabsf(x[u][i]));
          }
          m[u] = head_max<G>(finite ? most : INFINITY);
        }
        float mine = m[0];
#pragma unroll
        for (int u = 1; u < kHeads; u++) mine = sub == u ? m[u] : mine;
        const float dm = (float)((double)mine / 127.0);
        const double im = 1.0 / (double)dm;
#pragma unroll
        for (int u = 0; u < kHeads; u++) {
          d[u] = m[u] == INFINITY ? NAN : __shfl(dm, side * G + u);
          inv[u] = __shfl(im, side * G + u);
        }
      }
    }
    const int e_a = values ? 4 * sub : ea, e_b = values ? HD / 2 + 4 * sub : eb;
#pragma unroll
    for (int u = 0; u < kHeads; u++) {
      const int j = first + u * SIDE;
      if (j >= heads) continue;
      // four(element, values' index) or one(...) of the row
      auto put = [&](auto &&four, auto &&one) {
        if (ODD && !values) {
#pragma unroll
          for (int i = 0; i < 8; i++) one(e[ODD ? i : 0], i);
        } else {
          four(e_a, 0);
          four(e_b, 4);
        }
      };
      if (!values && j < a.heads) {
        float *o = a.q_out + (size_t)row * a.ld_out + (size_t)j * HD;
        if (bad) {
#pragma unroll
          for (int i = 0; i < 8; i++) x[u][i] = NAN;
        }
        put([&](int at, int i) {
          const f4u y = {x[u][i], x[u][i + 1], x[u][i + 2], x[u][i + 3]};
          // (MANY: past the caches, 45.6 -> 41.0 us with the read, of the keys and values
          // too 44.5; few rows stay for the attention that comes next)
          if constexpr (MANY) __builtin_nontemporal_store(y, reinterpret_cast<f4u *>(o + at));
          else *reinterpret_cast<f4u *>(o + at) = y;
        }, [&](int at, int i) { o[at] = x[u][i]; });
        continue;
      }
      if (bad) continue;
      const int64_t at = kv_row(a.kv, s, values, values ? j : j - a.heads, s.len + t);
      if constexpr (FMT == Q3H_KV_Q8) {
        uint8_t *o = reinterpret_cast<uint8_t *>(s.k0) + at * HD;
        const bool some = d[u] > 0.f;  // (not NaN, not 0)
        uint32_t y[8];
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = some ? byte_of(x[u][i], d[u], inv[u]) : 128;
        put([&](int at, int i) {
          *reinterpret_cast<uint32_t *>(o + at) =
              y[i] | y[i + 1] << 8 | y[i + 2] << 16 | y[i + 3] << 24;
        }, [&](int at, int i) { o[at] = y[i]; });
        if (sub == 0) kv_scales(a.kv, s, HD)[at] = d[u];
      } else {
        using KV = std::conditional_t<FMT == Q3H_KV_F16, _Float16, float>;
        typedef KV kv4 __attribute__((ext_vector_type(4)));
        KV *o = reinterpret_cast<KV *>(s.k0) + at * HD;
        put([&](int at, int i) {
          *reinterpret_cast<kv4 *>(o + at) =
              (kv4){to_cache<KV>(x[u][i]), to_cache<KV>(x[u][i + 1]), to_cache<KV>(x[u][i + 2]),
                    to_cache<KV>(x[u][i + 3])};
        }, [&](int at, int i) { o[at] = to_cache<KV>(x[u][i]); });
      }
    }
  }
}

// 4 elements of kReadRows rows per thread, keys then values. Memory bound: 32792
// positions of 8 heads of 128 from int8, 211 MB of which 168 are written, 34.7 us
// (6.1 TB/s). What it takes is that every store instruction writes whole lines, and
// past the caches: with 8 neighbouring elements a thread, half of each line an
// instruction, 57.8 us; through the caches 51.5. One row a thread 37.1, four 34.6.
constexpr int kReadRows = 2;
template <int FMT, int HD>
__global__ __launch_bounds__(kThreads) void k_cache_read(KvView kv, const int32_t *starts,
                                                         float *k, float *v) {
  constexpr int PER = HD / 4, SIDE = kThreads / PER;  // threads of a row, rows side by side
  using KV = std::conditional_t<FMT == Q3H_KV_F32, float,
                                std::conditional_t<FMT == Q3H_KV_F16, _Float16, uint8_t>>;
  typedef KV kv4 __attribute__((ext_vector_type(4)));
  typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
  const int e = (int)(threadIdx.x % PER) * 4;
  // the workgroup's first row (sequence, position, kv head)
  const int64_t r0 = (int64_t)blockIdx.x * (SIDE * kReadRows);
  const int64_t pos0 = r0 / kv.kvh;
  const int g0 = (int)(r0 - pos0 * kv.kvh), b0 = (int)(pos0 / kv.rows);
  const uint32_t t0 = (uint32_t)(pos0 - (int64_t)b0 * kv.rows);
  int64_t at[kReadRows];
  const char *base[kReadRows];
  bool there[kReadRows], bad[kReadRows];
#pragma unroll
  for (int u = 0; u < kReadRows; u++) {
    const uint32_t at0 = g0 + u * SIDE + threadIdx.x / PER;
    const uint32_t pos = at0 / (uint32_t)kv.kvh, g = at0 - pos * kv.kvh;
    const uint32_t over = (t0 + pos) / (uint32_t)kv.rows;
    const int b = b0 + (int)over, t = (int)(t0 + pos - over * kv.rows);
    const int in = min(b, kv.sequences - 1);
    KvSeq s;
    s.k0 = kv.base + in * kv.seq_bytes;
    s.max_pos = kv.max_pos;
    s.len = starts ? starts[in] : 0;
    s.count = kv.counts ? min(max(kv.counts[in], 0), kv.rows) : kv.rows;
    there[u] = b < kv.sequences && t < s.count;
    bad[u] = s.len < 0 || s.len > s.max_pos - s.count;
    // (no such row: the first one, which is there)
    at[u] = kv_row(kv, s, 0, there[u] ? (int)g : 0, there[u] && !bad[u] ? s.len + t : 0);
    base[u] = s.k0;
  }
  const int64_t values = (int64_t)kv.layers * kv.kvh * kv.max_pos;
#pragma unroll
  for (int part = 0; part < 2; part++) {
    float *dst = part ? v : k;
    if (!dst) continue;
    kv4 x[kReadRows];
    float d[kReadRows];
#pragma unroll
    for (int u = 0; u < kReadRows; u++) {
      const int64_t row = at[u] + part * values;
      x[u] = *reinterpret_cast<const kv4 *>(reinterpret_cast<const KV *>(base[u]) + row * HD + e);
      d[u] = FMT == Q3H_KV_Q8 ? reinterpret_cast<const float *>(base[u] + 2 * values * HD)[row] : 1.f;
    }
#pragma unroll
    for (int u = 0; u < kReadRows; u++) {
      if (!there[u]) continue;
      f4 o;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if constexpr (FMT == Q3H_KV_Q8) o[i] = kv_byte(x[u][i]) * d[u];
        else o[i] = (float)x[u][i];
        if (bad[u]) o[i] = NAN;
      }
      __builtin_nontemporal_store(
          o, reinterpret_cast<f4 *>(dst + (r0 + u * SIDE + threadIdx.x / PER) * HD + e));
    }
  }
}

// 32 sequences of 28 layers of 8 heads of 128, paths of 8 rows: f32 117 MB 29 us
// (4.1 TB/s), f16 26, int8 29; paths of 32 rows 179, 127 and 113 us; one sequence and
// a path of 8 5 us, of 32 12-16: bound by a trip to memory a row, one after another.
// One workgroup per (sequence, layer, kv head, keys or values): the kept rows
// in ascending order, each to a position at or before its own that no later
// row comes from, so one row after another is enough; a 4-byte word of a row a
// thread (HD = 64 int8: 16 words), the rest of the threads on the scale.
template <int FMT, int HD>
__global__ __launch_bounds__(128) void k_cache_keep(KvView kv, const int32_t *kept) {
  constexpr int WORDS = HD * (FMT == Q3H_KV_F32 ? 4 : FMT == Q3H_KV_F16 ? 2 : 1) / 4;
  const int b = blockIdx.x, tid = threadIdx.x;
  const KvSeq s = kv_sequence(kv, b);
  const int n = kv.counts[b];
  if (n < 1 || n > kv.rows || s.len < 0) return;
  const int32_t *list = kept + (size_t)b * kv.rows;
  // the list's form: ascending, in [0, rows), the last position inside the cache
  int last = -1;
  for (int i = 0; i < n; i++) {
    const int r = list[i];
    if (r <= last || r >= kv.rows) return;
    last = r;
  }
  if (s.len >= s.max_pos - last) return;
  const int layer = blockIdx.y / (2 * kv.kvh), lg = blockIdx.y - layer * 2 * kv.kvh;
  const int part = lg / kv.kvh, g = lg - part * kv.kvh;
  KvView at = kv;
  at.layer = layer;
  const int64_t first = kv_row(at, s, part, g, s.len);
  uint32_t *words = reinterpret_cast<uint32_t *>(s.k0) + first * WORDS;
  float *scales = kv_scales(at, s, HD) + first;
  for (int i = 0; i < n; i++) {
    const int r = list[i];
    if (r == i) continue;
    if (tid < WORDS) words[(int64_t)i * WORDS + tid] = words[(int64_t)r * WORDS + tid];
    if (FMT == Q3H_KV_Q8 && tid == WORDS) scales[i] = scales[r];
  }
}

// int8 rows from and to f32 [layers][kvh][len][HD], a wave a row
template <int HD>
__global__ void k_q8_fill(const float *src, char *k0, int part, int layers, int kvh, int len,
                          int max_pos) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (r >= (int64_t)layers * kvh * len) return;
  const int64_t lg = r / len, at = ((int64_t)part * layers * kvh + lg) * max_pos + (r - lg * len);
  float x[HD / 64], m = 0.f;
  bool finite = true;
#pragma unroll
  for (int e = 0; e < HD / 64; e++) {
    x[e] = src[r * HD + 64 * e + lane];
    finite = finite && fabsf(x[e]) < INFINITY;
    m = fmaxf(m, fabsf(x[e]));
  }
  m = wave_max_dpp(finite ? m : INFINITY);
  const float d = m == INFINITY ? NAN : (float)((double)m / 127.0);
  const double inv = 1.0 / (double)d;
#pragma unroll
  for (int e = 0; e < HD / 64; e++)
    reinterpret_cast<uint8_t *>(k0)[at * HD + 64 * e + lane] = d > 0.f ? byte_of(x[e], d, inv) : 128;
  if (lane == 0)
    reinterpret_cast<float *>(k0 + 2 * (int64_t)layers * kvh * max_pos * HD)[at] = d;
}
template <int HD>
__global__ void k_q8_read(const char *k0, int part, int layers, int layer, int kvh, int len,
                          int max_pos, float *dst) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (r >= (int64_t)kvh * len) return;
  const int64_t g = r / len;
  const int64_t at = (((int64_t)part * layers + layer) * kvh + g) * max_pos + (r - g * len);
  const float d = reinterpret_cast<const float *>(k0 + 2 * (int64_t)layers * kvh * max_pos * HD)[at];
#pragma unroll
  for (int e = 0; e < HD / 64; e++)
    dst[r * HD + 64 * e + lane] =
        kv_byte(reinterpret_cast<const uint8_t *>(k0)[at * HD + 64 * e + lane]) * d;
}

template <template <int, int> class F, class... A>
void by_format(int hd, int fmt, A &&...args) {
  if (hd == 64) {
    if (fmt == Q3H_KV_F32) F<Q3H_KV_F32, 64>::go(args...);
    else if (fmt == Q3H_KV_F16) F<Q3H_KV_F16, 64>::go(args...);
    else F<Q3H_KV_Q8, 64>::go(args...);
  } else {
    if (fmt == Q3H_KV_F32) F<Q3H_KV_F32, 128>::go(args...);
    else if (fmt == Q3H_KV_F16) F<Q3H_KV_F16, 128>::go(args...);
    else F<Q3H_KV_Q8, 128>::go(args...);
  }
}

template <int FMT, int HD>
struct GoAppend {
  static void go(const AppendRows &a, hipStream_t st) {
    const int per = kHeads * (512 / HD);  // heads of a wave at a time
    const int groups = (a.heads + a.kv.kvh + per - 1) / per + (a.kv.kvh + per - 1) / per;
    // few rows: a wave for each group of heads; many: one workgroup a row, its
    // waves going over the heads with one load of the angles
    const int rows = a.kv.sequences * a.kv.rows;
    const int side = rows >= kManyRows ? 1 : (groups + kThreads / 64 - 1) / (kThreads / 64);
    const dim3 grid(rows, side);
    if ((a.table || a.table32) && a.rot_dim % 8 != 0)
      hipLaunchKernelGGL((k_cache_append<FMT, HD, true, false>), grid, dim3(kThreads), 0, st, a);
    else if (rows >= kManyRows)
      hipLaunchKernelGGL((k_cache_append<FMT, HD, false, true>), grid, dim3(kThreads), 0, st, a);
    else
      hipLaunchKernelGGL((k_cache_append<FMT, HD, false, false>), grid, dim3(kThreads), 0, st, a);
  }
};
template <int FMT, int HD>
struct GoRead {
  static void go(const KvView &kv, const int32_t *starts, float *k, float *v, hipStream_t st) {
    const int64_t n = (int64_t)kv.sequences * kv.rows * kv.kvh, per = kReadRows * kThreads / (HD / 4);
    hipLaunchKernelGGL((k_cache_read<FMT, HD>), dim3((unsigned)((n + per - 1) / per)),
                       dim3(kThreads), 0, st, kv, starts, k, v);
  }
};
template <int FMT, int HD>
struct GoKeep {
  static void go(const KvView &kv, const int32_t *kept, hipStream_t st) {
    hipLaunchKernelGGL((k_cache_keep<FMT, HD>), dim3(kv.sequences, kv.layers * 2 * kv.kvh),
                       dim3(128), 0, st, kv, kept);
  }
};

// the pairs' angles per position, and the factor on cosine and sine
std::vector<double> rope_frequencies(const q3h_rope_config &c, double &mag) {
  const double pi = 3.14159265358979323846;
  const int pairs = c.rot_dim / 2;
  const double theta = c.theta, factor = c.factor, span = c.original_positions;
  std::vector<double> f(pairs);
  mag = 1.0;
  if (c.scaling == Q3H_ROPE_YARN && factor > 1.0) mag = 0.1 * std::log(factor) + 1.0;
  if (c.magnitude != 0.f) mag = c.magnitude;
  // the pair that turns `turns` times over the span
  auto pair_of = [&](double turns) {
    return c.rot_dim * std::log(span / (turns * 2.0 * pi)) / (2.0 * std::log(theta));
  };
  for (int i = 0; i < pairs; i++) {
    const double g = std::pow(theta, -2.0 * i / c.rot_dim);
    double own = 1.0;  // share of the unscaled frequency
    if (c.scaling == Q3H_ROPE_LINEAR) {
      own = 0.0;
    } else if (c.scaling == Q3H_ROPE_YARN) {
      const double lo = std::max(0.0, std::floor(pair_of(c.beta_fast)));
      const double hi = std::min(c.rot_dim - 1.0, std::ceil(pair_of(c.beta_slow)));
      own = 1.0 - std::min(1.0, std::max(0.0, (i - lo) / std::max(hi - lo, 0.001)));
    } else if (c.scaling == Q3H_ROPE_BANDS) {
      const double turns = span * g / (2.0 * pi);
      own = std::min(1.0, std::max(0.0, (turns - c.low_turns) / ((double)c.high_turns -
                                                                 (double)c.low_turns)));
    }
    f[i] = c.scaling == Q3H_ROPE_PLAIN ? g : g * own + g / factor * (1.0 - own);
  }
  return f;
}

// rows of pointers and row distances that every drafted-row call has
void check_rows(const q3h_cache *c, int layer, int sequences, int rows, const char *who) {
  const q3h_cache_config &f = c->cfg;
  if (layer < 0 || layer >= f.layers || sequences < 0 || sequences > f.sequences || rows < 0)
    require(false, Q3H_E_ARG,
            std::string(who) + ": layer " + std::to_string(layer) + ", " +
                std::to_string(sequences) + " sequences, " + std::to_string(rows) +
                " rows of a cache of " + std::to_string(f.layers) + " layers, " +
                std::to_string(f.sequences) + " sequences");
  if (rows > f.max_positions)
    require(false, Q3H_E_CAPACITY,
            std::string(who) + ": " + std::to_string(rows) + " rows in a cache of " +
                std::to_string(f.max_positions) + " positions");
}

// threads of a launch, below what a grid takes
bool launch_fits(int64_t blocks) { return blocks * kThreads < (int64_t)1 << 32; }

KvView view_of(const q3h_cache *c, int layer, int sequences, int rows, const int32_t *lens,
               const int32_t *counts) {
  KvView v{};
  v.base = c->data;
  v.seq_bytes = (int64_t)c->seq_bytes;
  v.lens = lens;
  v.counts = counts;
  v.layers = c->cfg.layers;
  v.kvh = c->cfg.kv_heads;
  v.max_pos = c->cfg.max_positions;
  v.layer = layer;
  v.sequences = sequences;
  v.rows = rows;
  return v;
}

}  // namespace

DeviceScope::DeviceScope(int ordinal) {
  int now = -1;
  check_hip(hipGetDevice(&now), "hipGetDevice");
  if (now == ordinal) return;
  check_hip(hipSetDevice(ordinal), "hipSetDevice");
  before_ = now;
}

DeviceScope::~DeviceScope() {
  if (before_ >= 0) (void)hipSetDevice(before_);
}

void launch_cache_append(const AppendRows &a, int hd, int fmt, hipStream_t st) {
  by_format<GoAppend>(hd, fmt, a, st);
}

void launch_cache_keep(const KvView &v, const int32_t *kept, int hd, int fmt, hipStream_t st) {
  by_format<GoKeep>(hd, fmt, v, kept, st);
}

void launch_q8_fill(const float *src, char *k0, bool values, int layers, int kvh, int len, int hd,
                    int max_pos, hipStream_t st) {
  const dim3 grid((unsigned)(((int64_t)layers * kvh * len + 3) / 4));
  if (hd == 64)
    hipLaunchKernelGGL(k_q8_fill<64>, grid, dim3(kThreads), 0, st, src, k0, values, layers, kvh,
                       len, max_pos);
  else
    hipLaunchKernelGGL(k_q8_fill<128>, grid, dim3(kThreads), 0, st, src, k0, values, layers, kvh,
                       len, max_pos);
}

void launch_q8_read(const char *k0, bool values, int layers, int layer, int kvh, int len, int hd,
                    int max_pos, float *dst, hipStream_t st) {
  const dim3 grid((unsigned)(((int64_t)kvh * len + 3) / 4));
  if (hd == 64)
    hipLaunchKernelGGL(k_q8_read<64>, grid, dim3(kThreads), 0, st, k0, values, layers, layer, kvh,
                       len, max_pos, dst);
  else
    hipLaunchKernelGGL(k_q8_read<128>, grid, dim3(kThreads), 0, st, k0, values, layers, layer,
                       kvh, len, max_pos, dst);
}

}  // namespace q3h

using namespace q3h;

// ---------------------------------------------------------------------------
// rotary tables

extern "C" int q3h_rope_create(q3h_device *dev, const q3h_rope_config *cfg, q3h_rope **out) {
  q3h_rope *r = nullptr;
  double *freq = nullptr;
  int rc = guard([&] {
    require(dev && cfg && out, Q3H_E_ARG, "q3h_rope_create: NULL argument");
    *out = nullptr;
    const q3h_rope_config &c = *cfg;
    require(c.head_dim == 64 || c.head_dim == 128, Q3H_E_ARG,
            "q3h_rope_create: head_dim must be 64 or 128");
    require(c.rot_dim >= 2 && c.rot_dim <= c.head_dim && c.rot_dim % 2 == 0, Q3H_E_ARG,
            "q3h_rope_create: rot_dim must be even and in [2, head_dim]");
    require(c.interleaved == 0 || c.interleaved == 1, Q3H_E_ARG,
            "q3h_rope_create: interleaved must be 0 or 1");
    require(c.max_positions > 0 && c.max_positions <= (1 << 24), Q3H_E_ARG,
            "q3h_rope_create: max_positions must be in [1, 2^24]");
    require(c.theta > 1.f && std::isfinite(c.theta), Q3H_E_ARG,
            "q3h_rope_create: theta must be above 1");
    require(c.scaling >= Q3H_ROPE_PLAIN && c.scaling <= Q3H_ROPE_BANDS, Q3H_E_ARG,
            "q3h_rope_create: no scaling " + std::to_string(c.scaling));
    require(c.scaling == Q3H_ROPE_PLAIN || (c.factor > 0.f && std::isfinite(c.factor)), Q3H_E_ARG,
            "q3h_rope_create: factor must be above 0");
    require(c.scaling < Q3H_ROPE_YARN || c.original_positions > 0, Q3H_E_ARG,
            "q3h_rope_create: original_positions must be above 0");
    require(c.scaling != Q3H_ROPE_YARN ||
                (c.beta_fast > c.beta_slow && c.beta_slow > 0.f && std::isfinite(c.beta_fast)),
            Q3H_E_ARG, "q3h_rope_create: beta_fast > beta_slow > 0 is needed");
    require(c.scaling != Q3H_ROPE_BANDS ||
                (c.high_turns > c.low_turns && c.low_turns > 0.f && std::isfinite(c.high_turns)),
            Q3H_E_ARG, "q3h_rope_create: high_turns > low_turns > 0 is needed");
    require(std::isfinite(c.magnitude) && c.magnitude >= 0.f, Q3H_E_ARG,
            "q3h_rope_create: magnitude must not be negative");
    DeviceScope scope(dev->ordinal);
    r = new q3h_rope();
    r->dev = dev;
    r->cfg = c;
    double mag = 1.0;
    const std::vector<double> f = rope_frequencies(c, mag);
    const size_t n = (size_t)c.max_positions * f.size();
    freq = (double *)dev_alloc(sizeof(double) * f.size());
    check_hip(hipMemcpy(freq, f.data(), sizeof(double) * f.size(), hipMemcpyHostToDevice),
              "upload frequencies");
    r->table = (double2 *)dev_alloc(sizeof(double2) * n);
    hipLaunchKernelGGL(k_rope_table, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, nullptr,
                       freq, mag, (int)f.size(), n, r->table);
    check_hip(hipGetLastError(), "rope table kernel");
    check_hip(hipStreamSynchronize(nullptr), "rope table sync");
    r->bytes = (int64_t)(sizeof(double2) * n);
    dev->bytes += r->bytes;
    dev->stacks++;
    *out = r;
  });
  dev_free(freq);
  if (rc != 0 && r) {
    dev_free(r->table);
    delete r;
  }
  return rc;
}

extern "C" int q3h_rope_destroy(q3h_rope *r) {
  return guard([&] {
    require(r != nullptr, Q3H_E_ARG, "q3h_rope_destroy: NULL table");
    DeviceScope scope(r->dev->ordinal);
    dev_free(r->table);
    r->dev->bytes -= r->bytes;
    r->dev->stacks--;
    delete r;
  });
}

// ---------------------------------------------------------------------------
// caches

extern "C" int q3h_cache_create(q3h_device *dev, const q3h_cache_config *cfg, q3h_cache **out) {
  q3h_cache *c = nullptr;
  int rc = guard([&] {
    require(dev && cfg && out, Q3H_E_ARG, "q3h_cache_create: NULL argument");
    *out = nullptr;
    require(cfg->sequences > 0 && cfg->layers > 0 && cfg->kv_heads > 0 && cfg->max_positions > 0,
            Q3H_E_ARG, "q3h_cache_create: non-positive dimension");
    require(cfg->sequences <= 65535 && cfg->kv_heads <= 1024 && cfg->layers <= 1024 &&
                cfg->max_positions <= (1 << 24) && (int64_t)cfg->layers * cfg->kv_heads <= 32767,
            Q3H_E_ARG, "q3h_cache_create: too many sequences, layers, heads or positions");
    require(cfg->head_dim == 64 || cfg->head_dim == 128, Q3H_E_ARG,
            "q3h_cache_create: head_dim must be 64 or 128");
    require(cfg->format >= Q3H_KV_F32 && cfg->format <= Q3H_KV_Q8, Q3H_E_ARG,
            "q3h_cache_create: format must be Q3H_KV_F32, Q3H_KV_F16 or Q3H_KV_Q8");
    DeviceScope scope(dev->ordinal);
    c = new q3h_cache();
    c->dev = dev;
    c->cfg = *cfg;
    const size_t need = kv_bytes(cfg->format, cfg->layers, cfg->kv_heads, cfg->max_positions,
                                 cfg->head_dim);
    c->seq_bytes = (need + 255) & ~(size_t)255;
    const size_t all = c->seq_bytes * cfg->sequences;
    c->data = (char *)dev_alloc(all);
    check_hip(hipMemset(c->data, 0, all), "zero cache");
    check_hip(hipStreamSynchronize(nullptr), "zero cache sync");
    c->bytes = (int64_t)all;
    dev->bytes += c->bytes;
    dev->stacks++;
    *out = c;
  });
  if (rc != 0 && c) {
    dev_free(c->data);
    delete c;
  }
  return rc;
}

extern "C" int64_t q3h_cache_bytes(const q3h_cache *c) { return c ? c->bytes : 0; }

extern "C" int q3h_cache_destroy(q3h_cache *c) {
  return guard([&] {
    require(c != nullptr, Q3H_E_ARG, "q3h_cache_destroy: NULL cache");
    DeviceScope scope(c->dev->ordinal);
    dev_free(c->data);
    c->dev->bytes -= c->bytes;
    c->dev->stacks--;
    delete c;
  });
}

extern "C" int q3h_cache_append(q3h_cache *c, const q3h_append_args *p, void *stream) {
  return guard([&] {
    require(c && p, Q3H_E_ARG, "q3h_cache_append: NULL argument");
    const q3h_cache_config &cf = c->cfg;
    check_rows(c, p->layer, p->sequences, p->rows, "q3h_cache_append");
    require(p->heads >= 0 && p->heads <= 4096, Q3H_E_ARG, "q3h_cache_append: bad heads");
    if (p->sequences == 0 || p->rows == 0) return;
    require(p->k && p->v && p->lens, Q3H_E_ARG, "q3h_cache_append: NULL k, v or lens");
    require(p->heads == 0 || (p->q && p->q_out), Q3H_E_ARG, "q3h_cache_append: NULL q or q_out");
    const int64_t wq = (int64_t)p->heads * cf.head_dim, wk = (int64_t)cf.kv_heads * cf.head_dim;
    require(p->ldk >= wk && p->ldv >= wk && (p->heads == 0 || (p->ldq >= wq && p->ld_out >= wq)),
            Q3H_E_ARG, "q3h_cache_append: rows overlap (a row distance below the row's width)");
    require(p->heads == 0 || p->q_out != p->q || p->ldq == p->ld_out, Q3H_E_ARG,
            "q3h_cache_append: in place with another row distance");
    require((p->q_norm == nullptr && p->k_norm == nullptr) || p->eps >= 0.f, Q3H_E_ARG,
            "q3h_cache_append: eps must not be negative");
    require(!p->parents || p->rows <= Q3H_TREE_MAX_ROWS, Q3H_E_CAPACITY,
            "q3h_cache_append: a tree has at most 64 rows");
    require(launch_fits((int64_t)p->sequences * p->rows), Q3H_E_CAPACITY,
            "q3h_cache_append: too many rows");
    if (p->rope) {
      require(p->rope->dev->ordinal == c->dev->ordinal, Q3H_E_ARG,
              "q3h_cache_append: rope of another device");
      require(p->rope->cfg.head_dim == cf.head_dim, Q3H_E_ARG,
              "q3h_cache_append: rope of another head_dim");
      require(p->rope->cfg.max_positions >= cf.max_positions, Q3H_E_ARG,
              "q3h_cache_append: the rope table has fewer positions than the cache");
    }
    DeviceScope scope(c->dev->ordinal);
    AppendRows a{};
    a.kv = view_of(c, p->layer, p->sequences, p->rows, p->lens, p->counts);
    a.heads = p->heads;
    a.q = p->q;
    a.k = p->k;
    a.v = p->v;
    a.ldq = p->ldq;
    a.ldk = p->ldk;
    a.ldv = p->ldv;
    a.q_out = p->q_out;
    a.ld_out = p->ld_out;
    a.q_norm = p->q_norm;
    a.k_norm = p->k_norm;
    a.eps = p->eps;
    if (p->rope) {
      a.table = p->rope->table;
      a.rot_dim = p->rope->cfg.rot_dim;
      a.interleaved = p->rope->cfg.interleaved;
    }
    a.parents = p->parents;
    launch_cache_append(a, cf.head_dim, cf.format, (hipStream_t)stream);
    check_hip(hipGetLastError(), "cache append kernel");
  });
}

extern "C" int q3h_cache_read(q3h_cache *c, int layer, int sequences, int rows,
                              const int32_t *starts, const int32_t *counts, float *k, float *v,
                              void *stream) {
  return guard([&] {
    require(c != nullptr, Q3H_E_ARG, "q3h_cache_read: NULL cache");
    check_rows(c, layer, sequences, rows, "q3h_cache_read");
    if (sequences == 0 || rows == 0 || (!k && !v)) return;
    const int64_t width = (int64_t)c->cfg.kv_heads * (c->cfg.head_dim / 8);  // threads a row
    require(launch_fits(((int64_t)sequences * rows * width + kThreads - 1) / kThreads),
            Q3H_E_CAPACITY, "q3h_cache_read: too many rows");
    DeviceScope scope(c->dev->ordinal);
    by_format<GoRead>(c->cfg.head_dim, c->cfg.format,
                      view_of(c, layer, sequences, rows, nullptr, counts), starts, k, v,
                      (hipStream_t)stream);
    check_hip(hipGetLastError(), "cache read kernel");
  });
}

extern "C" int q3h_cache_keep(q3h_cache *c, int sequences, int rows, const int32_t *lens,
                              const int32_t *kept, const int32_t *kept_counts, void *stream) {
  return guard([&] {
    require(c != nullptr, Q3H_E_ARG, "q3h_cache_keep: NULL cache");
    check_rows(c, 0, sequences, rows, "q3h_cache_keep");
    if (sequences == 0 || rows == 0) return;
    require(lens && kept && kept_counts, Q3H_E_ARG, "q3h_cache_keep: NULL argument");
    DeviceScope scope(c->dev->ordinal);
    launch_cache_keep(view_of(c, 0, sequences, rows, lens, kept_counts), kept, c->cfg.head_dim,
                      c->cfg.format, (hipStream_t)stream);
    check_hip(hipGetLastError(), "cache keep kernel");
  });
}

extern "C" int64_t q3h_cache_attend_workspace(const q3h_cache *c, int sequences, int rows,
                                              int heads, int max_len) {
  int64_t bytes = 0;
  const int rc = guard([&] {
    require(c != nullptr, Q3H_E_ARG, "q3h_cache_attend_workspace: NULL cache");
    check_rows(c, 0, sequences, rows, "q3h_cache_attend_workspace");
    require(heads > 0 && heads <= 4096 && heads % c->cfg.kv_heads == 0, Q3H_E_ARG,
            "q3h_cache_attend_workspace: heads must be a multiple of the cache's");
    require(max_len >= 0 && max_len <= c->cfg.max_positions, Q3H_E_ARG,
            "q3h_cache_attend_workspace: max_len beyond the cache");
    if (sequences == 0 || rows == 0) return;
    require(attend_fits(sequences, rows, heads, c->cfg.kv_heads, c->cfg.head_dim, c->cfg.format,
                        max_len),
            Q3H_E_CAPACITY, "q3h_cache_attend_workspace: too many rows, heads and positions");
    bytes = (int64_t)attend_part_bytes(sequences, rows, heads, c->cfg.kv_heads, c->cfg.head_dim,
                                       c->cfg.format, max_len);
  });
  return rc ? rc : bytes;
}

extern "C" int q3h_cache_attend(q3h_cache *c, const q3h_attend_args *p, void *stream) {
  return guard([&] {
    require(c && p, Q3H_E_ARG, "q3h_cache_attend: NULL argument");
    const q3h_cache_config &cf = c->cfg;
    check_rows(c, p->layer, p->sequences, p->rows, "q3h_cache_attend");
    require(p->heads > 0 && p->heads <= 4096 && p->heads % cf.kv_heads == 0, Q3H_E_ARG,
            "q3h_cache_attend: heads must be a multiple of the cache's");
    require(p->max_len >= 0 && p->max_len <= cf.max_positions, Q3H_E_ARG,
            "q3h_cache_attend: max_len beyond the cache");
    if (p->sequences == 0 || p->rows == 0) return;
    require(p->q && p->out && p->lens, Q3H_E_ARG, "q3h_cache_attend: NULL q, out or lens");
    const int64_t w = (int64_t)p->heads * cf.head_dim;
    require(p->ldq >= w && p->ld_out >= w, Q3H_E_ARG,
            "q3h_cache_attend: rows overlap (a row distance below the row's width)");
    require(p->out != p->q || p->ldq == p->ld_out, Q3H_E_ARG,
            "q3h_cache_attend: in place with another row distance");
    require(!p->parents || p->rows <= Q3H_TREE_MAX_ROWS, Q3H_E_CAPACITY,
            "q3h_cache_attend: a tree has at most 64 rows");
    require(attend_fits(p->sequences, p->rows, p->heads, cf.kv_heads, cf.head_dim, cf.format,
                        p->max_len),
            Q3H_E_CAPACITY, "q3h_cache_attend: too many rows, heads and positions");
    require(std::isfinite(p->scale), Q3H_E_ARG, "q3h_cache_attend: scale is not finite");
    const size_t need = attend_part_bytes(p->sequences, p->rows, p->heads, cf.kv_heads,
                                          cf.head_dim, cf.format, p->max_len);
    if (need > 0 && (!p->workspace || p->workspace_bytes < (int64_t)need ||
                     (uintptr_t)p->workspace % 256 != 0))
      require(false, Q3H_E_ARG, "q3h_cache_attend: a workspace of " + std::to_string(need) +
                                    " bytes, 256-byte aligned, is needed");
    DeviceScope scope(c->dev->ordinal);
    AttendRows a{};
    a.kv = view_of(c, p->layer, p->sequences, p->rows, p->lens, p->counts);
    a.heads = p->heads;
    a.max_len = p->max_len;
    a.scale = p->scale != 0.f ? p->scale : 1.0f / std::sqrt((float)cf.head_dim);
    a.q = p->q;
    a.ldq = p->ldq;
    a.out = p->out;
    a.ld_out = p->ld_out;
    a.parents = p->parents;
    a.part = (float *)p->workspace;
    a.room = need;
    launch_cache_attend(a, cf.head_dim, cf.format, (hipStream_t)stream);
    check_hip(hipGetLastError(), "cache attention kernels");
  });
}
