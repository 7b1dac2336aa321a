// q3h_score.hip - log probabilities of given tokens, the entropy of each row's
// distribution and its most likely tokens.
#include <hip/hip_runtime.h>

#include <string>

#include "q3h.h"
#include "q3h_api_internal.h"
#include "q3h_draft.h"
#include "q3h_wave.h"

namespace q3h {

namespace {

constexpr int kMaxVocab = 1 << 20;

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr float kLog2e = 1.44269504088896340736f;

// A logit as a number that orders it from the top: larger logits above, 0 and -0
// alike, NaN last; never 0. With its token's complement below it, as one 64-bit
// key, of equal logits the lower token is above, and no two keys are alike.
__device__ __forceinline__ uint32_t top_value(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 1u : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint64_t k) {
  const uint32_t v = (uint32_t)(k >> 32);
  if (v == 1u) return NAN;
  return __uint_as_float(v & 0x80000000u ? v & 0x7fffffffu : ~v);
}
__device__ __forceinline__ int key_token(uint64_t k) { return (int)~(uint32_t)k; }

// The k largest of the workgroup's keys (at most E a thread, key(e); 0: none),
// k <= 64: the k-th largest of the maxima of 64 groups of 4 threads is not
// above the k-th largest key, and only k groups hold keys from it on, so at
// most 4 k E keys are left (24 of 10240 on average for k = 20, 270 for 64); each
// of those counts the ones above it. emit(rank, key) once for every rank below
// min(k, keys).
struct TopSpace {
  union {
    uint64_t top[kThreads];
    float best[kThreads];
  };
  uint64_t bound;
  float value;
  int n;
};
// (the keys left: top_bytes of dynamic LDS)
inline size_t top_bytes(int k, int per_thread) {
  return (size_t)4 * k * per_thread * sizeof(uint64_t);
}
template <class Emit>
__device__ __forceinline__ void rank_list(const uint64_t *list, int n, int k, Emit &&emit) {
  for (int c = threadIdx.x; c < n; c += kThreads) {
    const uint64_t x = list[c];
    int rank = 0;
    for (int i = 0; i < n; i++) rank += list[i] > x;
    if (rank < k) emit(rank, x);
  }
}
template <int E, class Key, class Emit>
__device__ __forceinline__ void block_top(TopSpace &sm, uint64_t *list, int k, Key &&key, Emit &&emit) {
  const int tid = threadIdx.x, lane = tid & 63;
  uint64_t best = 0;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const uint64_t x = key(e);
    best = x > best ? x : best;
  }
  sm.top[tid] = best;
  if (tid == 0) sm.n = 0;
  __syncthreads();
  if (tid < 64) {
    uint64_t g = best;
#pragma unroll
    for (int i = 1; i < kWaves; i++) g = sm.top[64 * i + lane] > g ? sm.top[64 * i + lane] : g;
    int above = 0;
#pragma unroll
    for (int i = 0; i < 64; i++) {
      const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(g >> 32), i) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane((int)g, i);
      above += o > g;
    }
    // (one lane at most: no two keys alike)
    const uint64_t hit = __ballot(g && above == k - 1);
    if (hit == 0 ? lane == 0 : (hit >> lane & 1)) sm.bound = hit == 0 ? 1 : g;
  }
  __syncthreads();
  const uint64_t bound = sm.bound;
  if (best >= bound) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      const uint64_t x = key(e);
      if (x >= bound) list[atomicAdd(&sm.n, 1)] = x;
    }
  }
  __syncthreads();
  rank_list(list, sm.n, k, emit);
}

// The same for logits x(e), first by their values alone: the largest value that k
// of the 64 groups reach bounds the row's k-th from below, one comparison a logit.
// Where that leaves more than kShortList (many logits alike: a row of one value, or
// masked with a finite one down to fewer than k tokens) or bounds nothing (NaN,
// -infinity), by whole keys, which leave a few hundred of logits alike: ranks are
// counted for each key against all, 16.3 ms instead of 59 us for the top 64 of 40 rows
// of 151936 logits alike. best: the thread's largest logit.
constexpr int kShortList = 1024;
template <int E, class Logit, class Key, class Emit>
__device__ __forceinline__ void block_top_logits(TopSpace &sm, uint64_t *list, int k, float best,
                                                 Logit &&x, Key &&key, Emit &&emit) {
  const int tid = threadIdx.x, lane = tid & 63;
  sm.best[tid] = best;
  if (tid == 0) sm.n = 0;
  __syncthreads();
  if (tid < 64) {
    float g = best;
#pragma unroll
    for (int i = 1; i < kWaves; i++) g = fmaxf(g, sm.best[64 * i + lane]);
    int reach = 0;  // groups that reach this one's largest
#pragma unroll
    for (int i = 0; i < 64; i++) reach += lane_f(g, i) >= g;
    const float bound = wave_max_dpp(reach >= k ? g : -INFINITY);
    if (lane == 0) sm.value = bound;
  }
  __syncthreads();
  const float bound = sm.value;
  const int room = min(4 * k * E, kShortList);
  if (bound > -INFINITY) {
    if (best >= bound) {
      int n = 0;
#pragma unroll
      for (int e = 0; e < E; e++) n += x(e) >= bound;
      int at = atomicAdd(&sm.n, n);
      if (at + n <= room) {
#pragma unroll
        for (int e = 0; e < E; e++)
          if (x(e) >= bound) list[at++] = key(e);
      }
    }
    __syncthreads();
    const int n = sm.n;
    if (n <= room) {
      rank_list(list, n, k, emit);
      return;
    }
    __syncthreads();  // (sm.n is written again)
  }
  block_top<E>(sm, list, k, key, emit);
}

// A row's sums: the maximum, and over the logits' distances d from it the sums
// of e^d and of d e^d.
struct Sums {
  float m, s, u;
};

// what a row's sums and top tokens come to
__device__ __forceinline__ void finish_row(const ScoreRows &a, int r, const Sums &t, float ls) {
  for (int i = threadIdx.x; i < a.tokens_per_row; i += kThreads) {
    const int c = a.tokens[(size_t)r * a.tokens_per_row + i];
    float v = NAN;
    if (c >= 0 && c < a.vocab) {
      const size_t at = (size_t)r * a.ld + c;
      const float x =
          a.bf16 ? __uint_as_float((uint32_t) static_cast<const uint16_t *>(a.logits)[at] << 16)
                 : static_cast<const float *>(a.logits)[at];
      v = x - t.m - ls;
    }
    a.logprobs[(size_t)r * a.tokens_per_row + i] = v;
  }
  if (threadIdx.x == 0 && a.entropy) a.entropy[r] = ls - t.u / t.s;
}

// what a split of a row leaves for the merge: its sums, then top_k keys (0: none)
struct Space {
  Sums *sums;      // [rows][splits]
  uint64_t *keys;  // [rows][splits][top_k]
};
__host__ __device__ __forceinline__ size_t sums_bytes(int rows, int splits) {
  return ((size_t)rows * splits * sizeof(Sums) + 255) / 256 * 256;
}
__device__ __forceinline__ Space space_of(const ScoreRows &a, int splits) {
  Space s;
  s.sums = static_cast<Sums *>(a.work);
  s.keys = reinterpret_cast<uint64_t *>(static_cast<char *>(a.work) + sums_bytes(a.rows, splits));
  return s;
}

// One workgroup per (row, split of kThreads * E logits), the logits read once,
// 16 bytes a load, and kept in registers: the maximum, the sums, the top. Loads
// are at 16-byte boundaries whatever the row's: the row begins `skew` elements
// into its first.
//
// m = max x, s = sum e^(x - m), u = sum (x - m) e^(x - m): logprob = x - m - ln s,
// entropy = ln s - u / s. Bound by what a thread does with its logits (an
// exponential, two sums, two comparisons each) behind one round of loads, as
// all workgroups are on the chip at once: 1021 rows of 8191 bf16 logits, 16.8 MB,
// 12 us (17 with whole 64-bit keys compared for the top); 40 rows of 151936 f32
// logits, 24.3 MB in 600 workgroups, 12 us and the merge's 4.5; one row of 2048 4.4.
// 16 logits a thread for long rows were 5 % faster there and have three times the
// keys to merge: not kept. The list of keys is made for the most there can be (82 KB of
// LDS for the top 64 of 40 logits a thread, one workgroup a CU), and the bound comes
// down to the least of 64 groups: 40 rows of 151936 with the top 20 in 14 us, 33 in 15,
// 48 in 24, 64 in 104-115.
template <bool BF16, int E>
__global__ __launch_bounds__(kThreads) void k_score(ScoreRows a, int splits) {
  constexpr int VEC = BF16 ? 8 : 4, SIZE = BF16 ? 2 : 4;
  __shared__ TopSpace sm;
  extern __shared__ uint64_t list[];
  __shared__ float red[3][kWaves];
  const int r = blockIdx.x / splits, split = blockIdx.x - r * splits, tid = threadIdx.x;
  const char *row = static_cast<const char *>(a.logits) + (size_t)r * a.ld * SIZE;
  const int skew = (int)(reinterpret_cast<uintptr_t>(row) & 15) / SIZE;
  const int first = split * kThreads * E - skew + tid * VEC;  // the thread's first token
  float x[E];
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int v = 0; v < E / VEC; v++) {
    const int i = first + v * kThreads * VEC;
    float *y = x + v * VEC;
    if (i >= 0 && i + VEC <= a.vocab) {
      const u4 w = *reinterpret_cast<const u4 *>(row + (int64_t)i * SIZE);
#pragma unroll
      for (int e = 0; e < VEC; e++)
        y[e] = __uint_as_float(!BF16 ? w[e] : e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        y[e] = -INFINITY;
        if (i + e >= 0 && i + e < a.vocab)
          y[e] = BF16 ? __uint_as_float((uint32_t) reinterpret_cast<const uint16_t *>(row)[i + e]
                                        << 16)
                      : reinterpret_cast<const float *>(row)[i + e];
      }
    }
  }
  Sums t;
  t.m = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; e++) t.m = fmaxf(t.m, x[e]);
  const float best = t.m;
  t.m = wave_max_dpp(t.m);
  if ((tid & 63) == 0) red[0][tid >> 6] = t.m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; i++) t.m = fmaxf(t.m, red[0][i]);
  const float base = t.m == -INFINITY ? 0.f : t.m;
  t.s = t.u = 0.f;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const float d = x[e] - base, w = __builtin_amdgcn_exp2f(d * kLog2e);
    t.s += w;
    t.u = fmaf(fmaxf(d, -200.f), w, t.u);  // (w is 0 there, and not 0 * -infinity)
  }
  t.s = wave_sum_dpp(t.s);
  t.u = wave_sum_dpp(t.u);
  if ((tid & 63) == 0) {
    red[1][tid >> 6] = t.s;
    red[2][tid >> 6] = t.u;
  }
  __syncthreads();
  t.s = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  t.u = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
  const Space out = space_of(a, splits);
  const float ls = logf(t.s);
  if (splits == 1) finish_row(a, r, t, ls);
  else if (tid == 0) out.sums[blockIdx.x] = t;
  if (a.top_k == 0) return;
  uint64_t *keys = out.keys + (size_t)blockIdx.x * a.top_k;
  if (splits > 1 && tid < a.top_k && tid >= a.vocab - (split * kThreads * E - skew)) keys[tid] = 0;
  block_top_logits<E>(
      sm, list, a.top_k, best, [&](int e) { return x[e]; },
      [&](int e) -> uint64_t {
        const int i = first + e / VEC * kThreads * VEC + e % VEC;
        return i >= 0 && i < a.vocab ? (uint64_t)top_value(x[e]) << 32 | (uint32_t)~i : 0;
      },
      [&](int rank, uint64_t k) {
        if (splits == 1) {
          a.top_ids[(size_t)r * a.top_k + rank] = key_token(k);
          a.top_logprobs[(size_t)r * a.top_k + rank] = key_logit(k) - t.m - ls;
        } else {
          keys[rank] = k;
        }
      });
}

// The splits of a row together, a workgroup a row: 40 rows of 15 splits 4.5 us, a
// launch and three trips to memory (sums, keys, the given tokens' logits).
constexpr int kMergeKeys = 32;  // a thread, at most
template <int E>
__global__ __launch_bounds__(kThreads) void k_score_merge(ScoreRows a, int splits) {
  __shared__ TopSpace sm;
  extern __shared__ uint64_t list[];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const Space in = space_of(a, splits);
  const Sums *sums = in.sums + (size_t)r * splits;
  Sums t{-INFINITY, 0.f, 0.f};
  for (int i = lane; i < splits; i += 64) t.m = fmaxf(t.m, sums[i].m);
  t.m = wave_max_dpp(t.m);
  const float base = t.m == -INFINITY ? 0.f : t.m;
  for (int i = lane; i < splits; i += 64) {
    const Sums p = sums[i];
    const float d = p.m - base, f = __builtin_amdgcn_exp2f(d * kLog2e);
    if (p.s != 0.f) {  // (none: logits of -infinity alone)
      t.s += f * p.s;
      if (f != 0.f) t.u += f * (p.u + d * p.s);
    }
  }
  t.s = wave_sum_dpp(t.s);
  t.u = wave_sum_dpp(t.u);
  const float ls = logf(t.s);
  finish_row(a, r, t, ls);
  if (a.top_k == 0) return;
  const int n = splits * a.top_k;
  const uint64_t *keys = in.keys + (size_t)r * n;
  uint64_t mine[E];
#pragma unroll
  for (int e = 0; e < E; e++)
    mine[e] = e * kThreads + tid < n ? keys[e * kThreads + tid] : 0;
  block_top<E>(
      sm, list, a.top_k, [&](int e) { return mine[e]; },
      [&](int rank, uint64_t k) {
        a.top_ids[(size_t)r * a.top_k + rank] = key_token(k);
        a.top_logprobs[(size_t)r * a.top_k + rank] = key_logit(k) - t.m - ls;
      });
}

// Logits a thread: as few as cover the row with one workgroup, at most 40 (the
// registers of two workgroups a SIMD). A row that does not begin at a 16-byte
// boundary takes up to 7 more.
int score_width(int vocab) {
  return vocab + 7 <= kThreads * 8 ? 8 : vocab + 7 <= kThreads * 16 ? 16 : 40;
}
int score_splits(int vocab) {
  const int per = kThreads * score_width(vocab);
  return (vocab + 7 + per - 1) / per;
}
// a launch has fewer than 2^32 threads
bool score_fits(int rows, int vocab) {
  return (int64_t)rows * score_splits(vocab) * kThreads < (int64_t)1 << 32;
}
static_assert((kMaxVocab + 7 + kThreads * 40 - 1) / (kThreads * 40) * Q3H_TOP_MAX <=
                  kMergeKeys * kThreads,
              "the merge holds every split's keys");

template <bool BF16>
void launch(const ScoreRows &a, hipStream_t st) {
  const int splits = score_splits(a.vocab), width = score_width(a.vocab);
  const dim3 grid((unsigned)((int64_t)a.rows * splits));
  const size_t lds = top_bytes(a.top_k, width);
  if (width == 8)
    hipLaunchKernelGGL((k_score<BF16, 8>), grid, dim3(kThreads), lds, st, a, splits);
  else if (width == 16)
    hipLaunchKernelGGL((k_score<BF16, 16>), grid, dim3(kThreads), lds, st, a, splits);
  else
    hipLaunchKernelGGL((k_score<BF16, 40>), grid, dim3(kThreads), lds, st, a, splits);
  if (splits > 1) {
    const int keys = (splits * a.top_k + kThreads - 1) / kThreads;
    if (keys <= 2)
      hipLaunchKernelGGL((k_score_merge<2>), dim3(a.rows), dim3(kThreads), top_bytes(a.top_k, 2),
                         st, a, splits);
    else
      hipLaunchKernelGGL((k_score_merge<kMergeKeys>), dim3(a.rows), dim3(kThreads),
                         top_bytes(a.top_k, kMergeKeys), st, a, splits);
  }
}

}  // namespace

size_t score_work_bytes(int rows, int vocab, int top_k) {
  const int splits = score_splits(vocab);
  if (splits == 1) return 0;
  return sums_bytes(rows, splits) + (size_t)rows * splits * top_k * sizeof(uint64_t);
}

void launch_token_scores(const ScoreRows &a, hipStream_t st) {
  if (a.bf16) launch<true>(a, st);
  else launch<false>(a, st);
}

}  // namespace q3h

using namespace q3h;

extern "C" int64_t q3h_token_logprobs_workspace(int rows, int vocab, int top_k) {
  int64_t bytes = 0;
  const int rc = guard([&] {
    require(rows >= 0 && vocab > 0 && vocab <= kMaxVocab && top_k >= 0 && top_k <= Q3H_TOP_MAX && top_k <= vocab,
            Q3H_E_ARG, "q3h_token_logprobs_workspace: invalid argument");
    require(score_fits(rows, vocab), Q3H_E_CAPACITY,
            "q3h_token_logprobs_workspace: too many rows");
    if (rows > 0) bytes = (int64_t)score_work_bytes(rows, vocab, top_k);
  });
  return rc ? rc : bytes;
}

extern "C" int q3h_token_logprobs(q3h_device *dev, const q3h_score_args *p, void *stream) {
  return guard([&] {
    require(dev && p, Q3H_E_ARG, "q3h_token_logprobs: NULL argument");
    require(p->rows >= 0 && p->vocab > 0 && p->vocab <= kMaxVocab, Q3H_E_ARG,
            "q3h_token_logprobs: rows must not be negative, vocab in [1, 2^20]");
    require(p->dtype == Q3H_F32 || p->dtype == Q3H_BF16, Q3H_E_ARG,
            "q3h_token_logprobs: dtype must be Q3H_F32 or Q3H_BF16");
    require(p->tokens_per_row >= 0, Q3H_E_ARG, "q3h_token_logprobs: negative tokens_per_row");
    require(p->top_k >= 0 && p->top_k <= Q3H_TOP_MAX && p->top_k <= p->vocab, Q3H_E_ARG,
            "q3h_token_logprobs: top_k must be in [0, min(vocab, 64)]");
    if (p->rows == 0) return;
    require(p->logits != nullptr, Q3H_E_ARG, "q3h_token_logprobs: NULL logits");
    require((uintptr_t)p->logits % (p->dtype == Q3H_BF16 ? 2 : 4) == 0, Q3H_E_ARG,
            "q3h_token_logprobs: logits between elements");
    require(score_fits(p->rows, p->vocab), Q3H_E_CAPACITY, "q3h_token_logprobs: too many rows");
    require(p->ld >= p->vocab, Q3H_E_ARG, "q3h_token_logprobs: rows overlap (ld below vocab)");
    require(p->tokens_per_row == 0 || (p->tokens && p->logprobs), Q3H_E_ARG,
            "q3h_token_logprobs: NULL tokens or logprobs");
    require(p->top_k == 0 || (p->top_ids && p->top_logprobs), Q3H_E_ARG,
            "q3h_token_logprobs: NULL top_ids or top_logprobs");
    const size_t need = score_work_bytes(p->rows, p->vocab, p->top_k);
    if (need > 0 && (!p->workspace || p->workspace_bytes < (int64_t)need ||
                     (uintptr_t)p->workspace % 256 != 0))
      require(false, Q3H_E_ARG, "q3h_token_logprobs: a workspace of " + std::to_string(need) +
                                    " bytes, 256-byte aligned, is needed");
    DeviceScope scope(dev->ordinal);
    ScoreRows a{};
    a.logits = p->logits;
    a.ld = p->ld;
    a.bf16 = p->dtype == Q3H_BF16;
    a.rows = p->rows;
    a.vocab = p->vocab;
    a.tokens_per_row = p->tokens_per_row;
    a.top_k = p->top_k;
    a.tokens = p->tokens;
    a.logprobs = p->logprobs;
    a.entropy = p->entropy;
    a.top_ids = p->top_ids;
    a.top_logprobs = p->top_logprobs;
    a.work = p->workspace;
    launch_token_scores(a, (hipStream_t)stream);
    check_hip(hipGetLastError(), "token score kernels");
  });
}
