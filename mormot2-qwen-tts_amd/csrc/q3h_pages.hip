// q3h_pages.hip - the pages of a K/V cache that sequences share: reserving room for
// rows to come (with own copies of shared pages), forking sequences, releasing,
// moving the pages in use together, and copying sequences between caches.
//
// Which pages a sequence has is on the device (q3h_cache::state), so that a
// captured call follows it: table [sequences][slots] of page numbers (-1: none),
// held [sequences], how many of a row of it are there, refs [pages], how many
// sequences hold a page, 0: it is free. A page is taken lowest number first, the
// sequences in their order: the outcome does not depend on how the threads run.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "q3h.h"
#include "q3h_api_internal.h"
#include "q3h_draft.h"
#include "q3h_wave.h"

namespace q3h {

namespace {

constexpr int kThreads = 256, kBook = 1024, kBookWaves = kBook / 64;

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// The table and what a change of it needs, all in one allocation of 32-bit words.
// writers and lowest are 0 and kNobody between calls.
constexpr int kNobody = 0x7fffffff;
struct Book {
  int32_t *table, *held, *refs;
  int32_t *writers, *lowest;    // [pages]
  int32_t *order, *olds, *moved; // [pages]
  int32_t *next;                // [sequences][slots]: a fork's table
  int32_t *next_held;           // [sequences]
  int32_t *wanted;              // [sequences]
  int32_t *copy_from, *copy_to; // [sequences]
  int32_t *used, *moves, *come; // [1] each; come is 0 between calls
  int sequences, slots, pages, page_log2, max_pos;
};
__host__ __device__ inline size_t book_words(int sequences, int slots, int pages) {
  return 2 * (size_t)sequences * slots + 5 * (size_t)sequences + 6 * (size_t)pages + 3;
}
Book book_of(const q3h_cache *c) {
  const size_t n = c->cfg.sequences, slots = c->slots, pages = c->pages;
  Book k;
  k.table = c->state;
  k.held = k.table + n * slots;
  k.refs = k.held + n;
  k.writers = k.refs + pages;
  k.lowest = k.writers + pages;
  k.order = k.lowest + pages;
  k.olds = k.order + pages;
  k.moved = k.olds + pages;
  k.next = k.moved + pages;
  k.next_held = k.next + n * slots;
  k.wanted = k.next_held + n;
  k.copy_from = k.wanted + n;
  k.copy_to = k.copy_from + n;
  k.used = k.copy_to + n;
  k.moves = k.used + 1;
  k.come = k.used + 2;
  k.sequences = c->cfg.sequences;
  k.slots = c->slots;
  k.pages = c->pages;
  k.page_log2 = c->page_log2;
  k.max_pos = c->cfg.max_positions;
  return k;
}

// what other threads of the workgroup have changed by atomics
__device__ __forceinline__ int now(const int32_t *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void change(int32_t *p, int by) {
  __hip_atomic_fetch_add(p, by, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ int64_t lane_i64(int64_t x, int l) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32 |
                   (uint32_t)__builtin_amdgcn_readlane((int)x, l));
}
// inclusive sums over the lanes
__device__ __forceinline__ int64_t lane_sums64(int64_t x) {
#pragma unroll
  for (int i = 1; i < 64; i *= 2) {
    const int64_t y = __shfl_up((long long)x, i);
    if ((int)(threadIdx.x & 63) >= i) x += y;
  }
  return x;
}

// inclusive sums over the workgroup's threads, and the sum of all
__device__ __forceinline__ int book_sums(int x, int &all) {
  __shared__ int sm[kBookWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int here = wave_prefix_sum_i(x);
  __syncthreads();
  if (lane == 63) sm[wave] = here;
  __syncthreads();
  const int w = lane < kBookWaves ? sm[lane] : 0, upto = wave_prefix_sum_i(w);
  all = __builtin_amdgcn_readlane(upto, kBookWaves - 1);
  return here + (wave > 0 ? __builtin_amdgcn_readlane(upto, wave - 1) : 0);
}

__global__ void k_book_clear(Book k) {
  const size_t words = book_words(k.sequences, k.slots, k.pages);
  const size_t none = (size_t)k.sequences * k.slots, low = k.lowest - k.table;
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < words;
       i += (size_t)gridDim.x * blockDim.x)
    k.table[i] = i < none ? -1 : i >= low && i < low + k.pages ? kNobody : 0;
}

// what a sequence wants: slots first .. end - 1 to be written to, `held` there
struct Want {
  int first, end, held, len;
  bool bad;
};
__device__ __forceinline__ Want want_of(const Book &k, int b, int n, int rows, const int32_t *lens,
                                        const int32_t *counts) {
  Want w{0, 0, 0, 0, false};
  if (b >= n) return w;
  const int c = counts ? min(max(counts[b], 0), rows) : rows, page = 1 << k.page_log2;
  w.len = lens[b];
  w.held = k.held[b];
  w.bad = w.len < 0 || w.len > k.max_pos - c || w.len > (int64_t)w.held << k.page_log2;
  if (w.bad || c == 0) return w;
  w.first = w.len >> k.page_log2;
  w.end = (w.len + c - 1 + page) >> k.page_log2;
  return w;
}
__device__ __forceinline__ void mark_writer(const Book &k, int p, int b) {
  change(k.writers + p, 1);
  __hip_atomic_fetch_min(k.lowest + p, b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void forget(const Book &k, int p) {
  k.writers[p] = 0;
  k.lowest[p] = kNobody;
}

// The rows before lens of a page that is replaced, of one (layer, keys or values, kv
// head), by a wave, 4 KB at a time.
template <int FMT, int HD>
__device__ __forceinline__ void copy_tail(const KvView &v, int page, int from, int to, int rows,
                                          int section) {
  constexpr int ROW = kv_row_bytes(FMT, HD), AHEAD = 4;
  const int lane = threadIdx.x & 63;
  const int64_t all = 2 * (int64_t)v.layers * v.kvh * page, at = (int64_t)section * page;
  const char *src = v.base + from * v.seq_bytes;
  char *dst = v.base + to * v.seq_bytes;
  const u4 *x = reinterpret_cast<const u4 *>(src + at * ROW);
  u4 *y = reinterpret_cast<u4 *>(dst + at * ROW);
  // (a scale a row, and a word of steps)
  const uint32_t *sx = reinterpret_cast<const uint32_t *>(src + all * ROW) + at;
  uint32_t *sy = reinterpret_cast<uint32_t *>(dst + all * ROW) + at;
  const int chunks = rows * (ROW / 16);
  for (int i = lane; i < chunks; i += AHEAD * 64) {
    u4 r[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; j++) r[j] = x[min(i + j * 64, chunks - 1)];
#pragma unroll
    for (int j = 0; j < AHEAD; j++)
      if (i + j * 64 < chunks) y[i + j * 64] = r[j];
  }
  if constexpr (kv_scaled(FMT))
    for (int i = lane; i < rows; i += 64) {
      const uint32_t scale = sx[i], steps = FMT == Q3H_KV_Q4 ? sx[all + i] : 0;
      sy[i] = scale;
      if constexpr (FMT == Q3H_KV_Q4) sy[all + i] = steps;
    }
}

// The workgroups of a launch that all work out the same from the tables: true for the one
// that comes last, which alone may change them (the others have read what they need).
__device__ __forceinline__ bool last_to_come(const Book &k) {
  __shared__ int sm_last;
  __syncthreads();
  if (threadIdx.x == 0) {
    const int before = __hip_atomic_fetch_add(k.come, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sm_last = before == (int)gridDim.x - 1;
    if (sm_last) *k.come = 0;
  }
  __syncthreads();
  return sm_last;
}

// Pages for positions lens .. lens + counts - 1 of the first n sequences, where a thread
// each has a slot (`group` a sequence, a power of two up to 64, 1024 in all): what a thread
// finds stays in its registers, the writers of shared pages are counted in LDS, and the
// ranks of the pages taken are sums over the threads. Every workgroup does all that, copies
// its part of the rows before lens of the pages that are replaced, and the one that came
// last changes the tables: one launch. Bound by the trips to memory that wait for one
// another (lengths, table, holders) and the barriers, then by the copies: 4 sequences 5.3 us,
// 16 of up to 33 pages 5.6, four beams of a shared page 7.3 and 128 of 16 prompts, where the
// rows of 112 pages are copied in 5 layers of 4 bits, 29 MB read and written, 16.4. (In two
// launches, one workgroup and then the copies, fork and reserve of the four beams 16.8 us,
// 10.7 so.) At its largest, 1024 slots, it is still the faster form: 512 beams of 256 prompts
// 8 us (two launches 12), 64 sequences that take 15 pages each 8.3 with the release before
// (12.0); it is the threads and LDS that end there. Few free pages behind many used ones cost
// a scan by every workgroup: 16 pages, 99000 of 100000 in use, 54 us (57 in two launches).
template <int FMT, int HD>
__global__ __launch_bounds__(kBook) void k_reserve(Book k, KvView v, int n, int rows,
                                                   const int32_t *lens, const int32_t *counts,
                                                   int32_t *ok, int group) {
  constexpr int HASH = 2 * kBook;
  __shared__ int32_t sm_free[kBook], sm_key[HASH], sm_writers[HASH], sm_lowest[HASH];
  __shared__ int32_t sm_from[kBook], sm_to[kBook], sm_rows[kBook];
  const int tid = threadIdx.x, lane = tid & 63, page = 1 << k.page_log2;
  const int sub = lane & (group - 1), lane0 = lane & ~(group - 1), b = tid / group;
  const uint64_t lanes = group == 64 ? ~0ull : (1ull << group) - 1;
  constexpr int EACH = 8;
  auto is_free = [&](int p0, int i) {
    const int p = p0 + tid * EACH + i;
    return p < k.pages && k.refs[min(p, k.pages - 1)] == 0;
  };
  int mine[EACH];
#pragma unroll
  for (int i = 0; i < EACH; i++) mine[i] = is_free(0, i);
  const Want w = want_of(k, b, n, rows, lens, counts);
  const int at = w.first + sub;
  const bool in = at < w.end, there = in && at < w.held;
  int32_t *const slot = k.table + (size_t)min(b, n - 1) * k.slots + min(at, k.slots - 1);
  const int old = there ? *slot : -1, holders = there ? k.refs[old] : 0;
  const bool shared = holders > 1;
  bool take = in && !there;
  if (__syncthreads_or(shared)) {
    for (int i = tid; i < HASH; i += kBook) {
      sm_key[i] = -1;
      sm_writers[i] = 0;
      sm_lowest[i] = kNobody;
    }
    __syncthreads();
    int h = 0;
    if (shared) {
      // (at most 1024 pages for 2048 places)
      for (h = (int)((uint32_t)old * 2654435761u >> 21);; h = (h + 1) & (HASH - 1)) {
        const int was = atomicCAS(sm_key + h, -1, old);
        if (was == -1 || was == old) break;
      }
      atomicAdd(sm_writers + h, 1);
      atomicMin(sm_lowest + h, b);
    }
    __syncthreads();
    // (kept: by the first sequence, if all that hold a page write to it)
    if (shared) take = sm_writers[h] != holders || sm_lowest[h] != b;
  }
  int total, found = 0;
  const int upto = book_sums(take, total), r = upto - take;
  // the lowest free pages
  for (int p0 = 0; p0 < k.pages && found < total; p0 += kBook * EACH) {
    int free = 0, all;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      if (p0 > 0) mine[i] = is_free(p0, i);
      free += mine[i];
    }
    int rank = found + book_sums(free, all) - free;
#pragma unroll
    for (int i = 0; i < EACH; i++)
      if (mine[i]) {
        if (rank < total) sm_free[rank] = p0 + tid * EACH + i;
        rank++;
      }
    found += all;
  }
  const uint64_t takes = __ballot(take) >> lane0 & lanes;
  const int wanted = __popcll(takes), last = __shfl(upto, lane0 + group - 1);
  const bool gets = wanted == 0 || last <= found;
  const bool changes = last_to_come(k);  // (a barrier: sm_free is whole)
  const int fresh = take && gets ? sm_free[r] : -1;
  if (sub == 0) {
    // (the group's first lane has the first slot)
    const int tail = fresh >= 0 && old >= 0 ? w.len & (page - 1) : 0;
    sm_from[b] = old;
    sm_to[b] = fresh;
    sm_rows[b] = tail;
  }
  if (changes) {
    if (fresh >= 0) {
      *slot = fresh;
      k.refs[fresh] = 1;
      if (old >= 0) change(k.refs + old, -1);
    }
    if (b < n && sub == 0 && gets && wanted > 0 && w.end > w.held) k.held[b] = w.end;
    if (ok) {
      __syncthreads();
      // (a shared page that it keeps is its own if all others have left it)
      const uint64_t others =
          __ballot(shared && fresh < 0 && now(k.refs + old) > 1) >> lane0 & lanes;
      if (b < n && sub == 0) ok[b] = !w.bad && gets && others == 0;
    }
  }
  __syncthreads();
  const int sections = 2 * v.layers * v.kvh, waves = gridDim.x * kBookWaves;
  for (int i = blockIdx.x * kBookWaves + __builtin_amdgcn_readfirstlane(tid >> 6); i < n * sections;
       i += waves) {
    const int s = i / sections;
    if (sm_rows[s] > 0) copy_tail<FMT, HD>(v, page, sm_from[s], sm_to[s], sm_rows[s], i - s * sections);
  }
}

// The same of any number of slots, and a launch for the copies: one workgroup, `group`
// lanes (a power of two) a sequence at a time: who writes to which shared page (writers,
// lowest), how many pages each sequence wants, their sums in order, the lowest free pages in
// order, who gets which. A pass over the slots for each, of one workgroup's trips to memory:
// 32 sequences of up to 64 pages at once 13.3 us, 1024 beams of 512 prompts 17.5 with the
// copies, 2048 of 1024 30, 256 sequences of 15 pages that they have already 16.7.
__global__ __launch_bounds__(kBook) void k_reserve_many(Book k, int n, int rows, const int32_t *lens,
                                                        const int32_t *counts, int32_t *ok,
                                                        int group) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int sub = lane & (group - 1), lane0 = lane & ~(group - 1);
  const uint64_t lanes = group == 64 ? ~0ull : (1ull << group) - 1;
  const int page = 1 << k.page_log2;
  // f(sequence, what it wants, slot, whether it is one of those) with all lanes of a wave
  auto each = [&](auto &&f) {
    for (int b0 = 0; b0 < n; b0 += kBook / group) {
      const int b = b0 + tid / group;
      const Want w = want_of(k, b, n, rows, lens, counts);
      int at = w.first + sub;
      do {
        f(b, w, at, at < w.end);
        at += group;
      } while (__any(at - sub < w.end));
    }
  };
  auto row = [&](int b, int at) { return k.table + (size_t)b * k.slots + at; };
  each([&](int b, const Want &w, int at, bool in) {
    if (in && at < w.held) {
      const int p = *row(b, at);
      if (k.refs[p] > 1) mark_writer(k, p, b);
    }
  });
  __syncthreads();
  // (kept: by the first sequence, if all that hold a page write to it)
  int sum = 0;
  each([&](int b, const Want &w, int at, bool in) {
    bool take = in && at >= w.held;
    if (in && at < w.held) {
      const int p = *row(b, at), writers = now(k.writers + p);
      if (writers > 0) {
        const bool all = writers == k.refs[p];
        take = !all || now(k.lowest + p) != b;
        if (!all) k.lowest[p] = -1;
      }
    }
    const int here = __popcll(__ballot(take) >> lane0 & lanes);
    sum = at == w.first + sub ? here : sum + here;
    if (sub == 0 && b < n) k.wanted[b] = sum;
  });
  __syncthreads();
  // the pages wanted before each sequence
  int total = 0;
  for (int b0 = 0; b0 < n; b0 += kBook) {
    const int b = b0 + tid, x = b < n ? k.wanted[b] : 0;
    int all;
    const int upto = book_sums(x, all);
    if (b < n) k.next_held[b] = total + upto - x;
    total += all;
  }
  // the lowest free pages
  int found = 0;
  constexpr int EACH = 8;
  for (int p0 = 0; p0 < k.pages && found < total; p0 += kBook * EACH) {
    int free = 0, mine[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const int p = p0 + tid * EACH + i;
      mine[i] = p < k.pages && k.refs[min(p, k.pages - 1)] == 0;
      free += mine[i];
    }
    int all;
    int at = found + book_sums(free, all) - free;
#pragma unroll
    for (int i = 0; i < EACH; i++)
      if (mine[i]) {
        if (at < total) k.order[at] = p0 + tid * EACH + i;
        at++;
      }
    found += all;
  }
  __syncthreads();
  sum = 0;
  each([&](int b, const Want &w, int at, bool in) {
    const bool start = at == w.first + sub;
    if (start) sum = b < n ? k.next_held[b] : 0;
    const int wanted = b < n ? k.wanted[b] : 0, before = b < n ? k.next_held[b] : 0;
    const bool gets = wanted > 0 && before + wanted <= found;
    int old = -1;
    bool take = in && at >= w.held;
    if (in && at < w.held) {
      const int p = *row(b, at);
      if (now(k.writers + p) > 0 && now(k.lowest + p) != b) {
        take = true;
        old = p;
      }
    }
    const uint64_t mask = __ballot(take) >> lane0 & lanes;
    const int r = sum + __popcll(mask & ((1ull << sub) - 1));
    sum += __popcll(mask);
    if (start && sub == 0 && b < n) k.copy_from[b] = -1;
    if (take && gets) {
      const int p = k.order[r];
      *row(b, at) = p;
      k.refs[p] = 1;
      k.olds[r] = old;
      if (old >= 0) {
        change(k.refs + old, -1);
        if (at == w.first && (w.len & (page - 1)) > 0) {
          // (its own lane of the group's first)
          k.copy_from[b] = old;
          k.copy_to[b] = p;
        }
      }
    }
    if (gets && start && sub == 0 && w.end > w.held) k.held[b] = w.end;
  });
  __syncthreads();
  // what the call has counted is forgotten; whether a sequence has its pages to itself
  bool shared = false;
  each([&](int b, const Want &w, int at, bool in) {
    const bool start = at == w.first + sub;
    if (start) shared = false;
    const int wanted = b < n ? k.wanted[b] : 0, before = b < n ? k.next_held[b] : 0;
    const bool gets = before + wanted <= found || wanted == 0;
    // (w.held is the new number where pages were taken)
    const bool there = in && at < (b < n ? k.held[b] : 0);
    bool others = false;
    if (there) {
      const int p = *row(b, at);
      forget(k, p);
      others = now(k.refs + p) > 1;
    }
    if (gets && b < n)
      for (int r = before + (start ? sub : wanted); r < before + wanted; r += group)
        if (k.olds[r] >= 0) forget(k, k.olds[r]);
    shared = shared || (__ballot(others) >> lane0 & lanes) != 0;
    if (ok && b < n && sub == 0) ok[b] = !w.bad && gets && !shared;
  });
}

template <int FMT, int HD>
__global__ __launch_bounds__(kThreads) void k_copy_tails(KvView v, Book k, const int32_t *lens) {
  const int b = blockIdx.x, from = k.copy_from[b];
  const int section = blockIdx.y * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (from < 0 || section >= 2 * v.layers * v.kvh) return;
  const int page = 1 << k.page_log2;
  copy_tail<FMT, HD>(v, page, from, k.copy_to[b], lens[b] & (page - 1), section);
}

// A fork's table: of up to 4096 entries (and 1024 sequences) by one workgroup, four of them a
// thread in registers between reading and writing (an assignment may be any, so that none is
// written before all are read); of more in two launches, the table beside the present one
// first. A chain of four trips to memory, in a graph: 4 sequences of two slots 2.6 us (two
// launches 5.0), 128 of 16 3.4 (5.2), 1024 of 4 4.2 (5.7), 64 of 64 4.1 (5.1), 256 of 17 in
// two 5.4. With sixteen entries a thread, each asked for in turn, 64 of two took 4.1 us, and
// 512 of 32 in one launch 10.0 (two 5.2).
constexpr int kForkEach = 4, kForkSlots = kForkEach * kBook;
struct Forked {
  int from, now, held;  // (now < 0: as it is)
};
__device__ __forceinline__ Forked forked(const Book &k, int b, const int32_t *sources,
                                         const int32_t *lens) {
  Forked f{sources[b], 0, k.held[b]};
  if (f.from >= 0 && f.from < k.sequences) {
    const int len = lens[b], held = k.held[f.from];
    // (the last page can reach behind the cache's positions)
    f.now = len < 0 || len > k.max_pos || len > (int64_t)held << k.page_log2
                ? -1
                : (int)(((int64_t)len + (1 << k.page_log2) - 1) >> k.page_log2);
  } else if (f.from != -1) {
    f.now = -1;
  }
  return f;
}
__device__ __forceinline__ void hold(const Book &k, int was, int is) {
  if (is == was) return;
  if (is >= 0) change(k.refs + is, 1);
  if (was >= 0) change(k.refs + was, -1);
}
__global__ __launch_bounds__(kBook) void k_fork_few(Book k, int n, const int32_t *sources,
                                                    const int32_t *lens) {
  __shared__ Forked sm[kBook];
  const int tid = threadIdx.x;
  if (tid < n) sm[tid] = forked(k, tid, sources, lens);
  __syncthreads();
  int is[kForkEach], was[kForkEach];
#pragma unroll
  for (int j = 0; j < kForkEach; j++) {
    const int i = tid + j * kBook, b = i / k.slots, at = i - b * k.slots;
    is[j] = was[j] = -1;
    if (b >= n) continue;
    const Forked f = sm[b];
    if (f.now < 0) continue;
    if (at < f.held) was[j] = k.table[i];
    if (at < f.now) is[j] = k.table[(size_t)f.from * k.slots + at];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kForkEach; j++) {
    if (is[j] == was[j]) continue;
    hold(k, was[j], is[j]);
    k.table[tid + j * kBook] = is[j];
  }
  if (tid < n && sm[tid].now >= 0) k.held[tid] = sm[tid].now;
}
__global__ __launch_bounds__(kThreads) void k_fork(Book k, const int32_t *sources,
                                                   const int32_t *lens) {
  const int b = blockIdx.x;
  const Forked f = forked(k, b, sources, lens);
  if (threadIdx.x == 0) k.next_held[b] = f.now;
  const int32_t *row = k.table + (size_t)b * k.slots,
                *src = k.table + (size_t)max(f.from, 0) * k.slots;
  for (int i = threadIdx.x; f.now >= 0 && i < max(f.now, f.held); i += kThreads) {
    const int was = i < f.held ? row[i] : -1, is = i < f.now ? src[i] : -1;
    k.next[(size_t)b * k.slots + i] = is;
    hold(k, was, is);
  }
}
__global__ __launch_bounds__(kThreads) void k_fork_end(Book k) {
  const int b = blockIdx.x, n = k.next_held[b], held = k.held[b];
  if (n < 0) return;
  for (int i = threadIdx.x; i < max(n, held); i += kThreads)
    k.table[(size_t)b * k.slots + i] = k.next[(size_t)b * k.slots + i];
  __syncthreads();
  if (threadIdx.x == 0) k.held[b] = n;
}

__global__ __launch_bounds__(64) void k_release(Book k, const int32_t *lens) {
  const int b = blockIdx.x, len = lens[b], held = k.held[b];
  if (len < 0) return;
  const int n = min(held, (int)(((int64_t)len + (1 << k.page_log2) - 1) >> k.page_log2));
  int32_t *row = k.table + (size_t)b * k.slots;
  for (int i = n + threadIdx.x; i < held; i += 64) {
    change(k.refs + row[i], -1);
    row[i] = -1;
  }
  if (threadIdx.x == 0) k.held[b] = n;
}

// Which pages move: the k-th of those in use behind their number to the k-th free one
// below it. list(k-th, page, whether it moves); returns the pages in use and how many move.
constexpr int kScan = 8 * kBook;
template <class F>
__device__ __forceinline__ int2 compact_lists(const Book &k, F &&list) {
  const int tid = threadIdx.x;
  constexpr int EACH = kScan / kBook;
  int in_use = 0, held[EACH];
  for (int p0 = 0; p0 < k.pages; p0 += kScan) {
    int here = 0, all;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const int p = p0 + tid * EACH + i;
      held[i] = k.refs[min(p, k.pages - 1)];
      here += p < k.pages && held[i] > 0;
    }
    book_sums(here, all);
    in_use += all;
  }
  int holes = 0, movers = 0;
  for (int p0 = 0; p0 < k.pages; p0 += kScan) {
    int here = 0, all, kind[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const int p = p0 + tid * EACH + i;
      if (k.pages > kScan) held[i] = k.refs[min(p, k.pages - 1)];
      // (a hole counts 1, a mover 2^16: 8192 pages at a time)
      kind[i] = p >= k.pages ? 0 : p < in_use ? held[i] <= 0 : held[i] > 0 ? 1 << 16 : 0;
      here += kind[i];
    }
    const int upto = book_sums(here, all) - here;
    int hole = holes + (upto & 0xffff), mover = movers + (upto >> 16);
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      if (kind[i] == 1) list(hole++, p0 + tid * EACH + i, false);
      if (kind[i] == 1 << 16) list(mover++, p0 + tid * EACH + i, true);
    }
    holes += all & 0xffff;
    movers += all >> 16;
  }
  return make_int2(in_use, movers);
}
// the contents of pages from[i] to pages to[i], by `all` threads of a launch
template <int AHEAD>
__device__ __forceinline__ void move_pages(char *base, int64_t page_bytes, int moves,
                                           const int32_t *from, const int32_t *to, int64_t first,
                                           int64_t step) {
  const int64_t per = page_bytes / 16, all = moves * per;
  for (int64_t i = first; i < all; i += AHEAD * step) {
    u4 x[AHEAD];
    u4 *dst[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; j++) {
      const int64_t at = min(i + j * step, all - 1), m = at / per, off = at - m * per;
      dst[j] = reinterpret_cast<u4 *>(base + to[m] * page_bytes) + off;
      x[j] = reinterpret_cast<const u4 *>(base + from[m] * page_bytes)[off];
    }
#pragma unroll
    for (int j = 0; j < AHEAD; j++)
      if (i + j * step < all) *dst[j] = x[j];
  }
}

// Up to 8192 pages: every workgroup works out the moves, makes its part of them and of
// the tables' changes, and the last to come changes who holds which page. Nothing to move:
// 6.4 us, a scan of all pages by every workgroup before its first load; 164 of 64 positions
// and 2 layers of int8, 89 MB read and written, 20. Against one workgroup and a launch for the
// moves, with few workgroups (pages of 2.5 KB, nothing to move / half of them): 1024 pages 4.6
// / 7.5 us (5.9 / 7.5), 4096 6.5 / 9.6 (7.1 / 11.7), 8192 9.2 / 13.8 (8.7 / 16.2); with 512
// of them nothing to move of 512 pages of 7.3 MB 10.0 (5.6) and of 8192 of 135 KB 13.7 (8.7),
// half of the 512 moved, 3.8 GB read and written, 774 (791). What moves in earnest decides for
// one launch; the lists in LDS end at 8192.
__global__ __launch_bounds__(kBook) void k_compact(Book k, char *base, int64_t page_bytes,
                                                   int32_t *used) {
  __shared__ int32_t sm_hole[kScan / 2], sm_mover[kScan / 2];
  const int tid = threadIdx.x;
  // (of as many holes below the number in use as there are movers behind it, at most half
  // of the pages)
  const int2 n = compact_lists(k, [&](int i, int p, bool moves) { (moves ? sm_mover : sm_hole)[i] = p; });
  const int in_use = n.x, moves = n.y;
  if (last_to_come(k)) {
    for (int i = tid; i < moves; i += kBook) {
      k.refs[sm_hole[i]] = k.refs[sm_mover[i]];
      k.refs[sm_mover[i]] = 0;
    }
    if (used && tid == 0) *used = in_use;
  }
  if (moves == 0) return;
  const int lane = tid & 63;
  const int waves = gridDim.x * kBookWaves;
  for (int b = blockIdx.x * kBookWaves + (tid >> 6); b < k.sequences; b += waves) {
    const int held = k.held[b];
    int32_t *row = k.table + (size_t)b * k.slots;
    for (int i = lane; i < held; i += 64) {
      const int p = row[i];
      if (p < in_use) continue;
      // (its place among the movers, which are in order)
      int lo = 0, hi = moves - 1;
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (sm_mover[mid] < p) lo = mid + 1;
        else hi = mid;
      }
      row[i] = sm_hole[lo];
    }
  }
  move_pages<4>(base, page_bytes, moves, sm_mover, sm_hole, (int64_t)blockIdx.x * kBook + tid,
                (int64_t)gridDim.x * kBook);
}

// Any number of pages: one workgroup for the lists, a mover's new place in moved, then the
// moves and the tables of the sequences. The scan of the holders is the time: 16384 pages,
// nothing to move, 20 us, 100000 101.
__global__ __launch_bounds__(kBook) void k_compact_many(Book k, int32_t *used) {
  const int2 n = compact_lists(k, [&](int i, int p, bool moves) { (moves ? k.order : k.olds)[i] = p; });
  __syncthreads();
  for (int i = threadIdx.x; i < n.y; i += kBook) {
    const int from = k.order[i], to = k.olds[i];
    k.moved[from] = to;
    k.refs[to] = k.refs[from];
    k.refs[from] = 0;
  }
  if (threadIdx.x == 0) {
    *k.used = n.x;
    *k.moves = n.y;
    if (used) *used = n.x;
  }
}
__global__ __launch_bounds__(kThreads) void k_move(Book k, char *base, int64_t page_bytes) {
  const int moves = *k.moves, in_use = *k.used;
  for (int b = blockIdx.x; b < k.sequences && moves > 0; b += gridDim.x) {
    const int held = k.held[b];
    int32_t *row = k.table + (size_t)b * k.slots;
    for (int i = threadIdx.x; i < held; i += kThreads) {
      const int p = row[i];
      if (p >= in_use) row[i] = k.moved[p];
    }
  }
  move_pages<4>(base, page_bytes, moves, k.order, k.olds, (int64_t)blockIdx.x * kThreads + threadIdx.x,
                (int64_t)gridDim.x * kThreads);
}

// The first lens[b] positions of sequence sources[b] of a cache into sequence b of
// another. A wave takes runs of 32 positions of a (layer, part, kv head), which lie in
// one piece on both sides, an equal share of all of them. 8 sequences, 10300
// positions of 2 layers of int8, 87 MB read and written: 19 us (4.6 TB/s).
template <int FMT, int HD>
__global__ __launch_bounds__(kThreads) void k_copy(KvView to, KvView from, const int32_t *sources,
                                                   int src_sequences) {
  constexpr int ROW = kv_row_bytes(FMT, HD), RUN = 32, LOADS = RUN * ROW / 1024 > 0 ? RUN * ROW / 1024 : 1;
  const int lane = threadIdx.x & 63;
  const int64_t worker = (int64_t)blockIdx.x * (kThreads / 64) +
                         __builtin_amdgcn_readfirstlane(threadIdx.x >> 6),
                workers = (int64_t)gridDim.x * (kThreads / 64);
  const int n = to.sequences, sections = 2 * to.layers * to.kvh;
  // what is copied of a sequence, 0 where that is not to be
  auto length = [&](int b) {
    if (b >= n) return 0;
    const int src = sources[b], len = to.lens[b];
    if (src < 0 || src >= src_sequences || len < 0) return 0;
    const int room = to.table ? kv_room(to, b) : to.max_pos;
    const int have = from.table ? kv_room(from, src) : from.max_pos;
    return len > room || len > have ? 0 : len;
  };
  auto copy_run = [&](int b, int section, int run, int len) {
    const int rows = min(RUN, len - run * RUN);
    int p = run * RUN, q = p;
    int64_t dst_at = b, src_at = sources[b];
    if (to.table) {
      dst_at = kv_page(to, b, p >> to.page_log2);
      if (to.refs[dst_at] > 1) return;  // (another sequence's too)
      p &= (1 << to.page_log2) - 1;
    }
    if (from.table) {
      src_at = kv_page(from, (int)src_at, q >> from.page_log2);
      q &= (1 << from.page_log2) - 1;
    }
    const int64_t to_each = to.table ? 1 << to.page_log2 : to.max_pos,
                  from_each = from.table ? 1 << from.page_log2 : from.max_pos;
    char *dst = to.base + dst_at * to.seq_bytes;
    const char *src = from.base + src_at * from.seq_bytes;
    const int64_t y = section * to_each + p, x = section * from_each + q;
    const u4 *sx = reinterpret_cast<const u4 *>(src + x * ROW);
    u4 *sy = reinterpret_cast<u4 *>(dst + y * ROW);
    const int chunks = rows * (ROW / 16);
    u4 r[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++) r[i] = sx[min(i * 64 + lane, chunks - 1)];
    uint32_t scale = 0;
    const uint32_t *cx = reinterpret_cast<const uint32_t *>(src + sections * from_each * ROW) + x;
    uint32_t *cy = reinterpret_cast<uint32_t *>(dst + sections * to_each * ROW) + y;
    // (scales in the lower half of the wave, steps in the upper one)
    const bool low = lane < 32;
    const int c = lane & 31;
    const bool has = kv_scaled(FMT) && c < rows && (low || FMT == Q3H_KV_Q4);
    if (has) scale = cx[(low ? 0 : sections * from_each) + c];
#pragma unroll
    for (int i = 0; i < LOADS; i++)
      if (i * 64 + lane < chunks) sy[i * 64 + lane] = r[i];
    if (has) cy[(low ? 0 : sections * to_each) + c] = scale;
  };
  auto runs_of = [&](int len) { return (int64_t)((len + RUN - 1) / RUN) * sections; };
  int64_t all = 0;
  for (int base = 0; base < n; base += 64) all += lane_i64(lane_sums64(runs_of(length(base + lane))), 63);
  int64_t item = all * worker / workers, before = 0;
  const int64_t end = all * (worker + 1) / workers;
  for (int base = 0; base < n && item < end; base += 64) {
    // 64 sequences in the lanes
    const int mine = length(base + lane);
    const int64_t upto = before + lane_sums64(runs_of(mine));
    before = lane_i64(upto, 63);
    while (item < end && item < before) {
      const int f = __builtin_ctzll(__ballot(upto > item));
      const int b = base + f, len = __builtin_amdgcn_readlane(mine, f);
      const int64_t stop = lane_i64(upto, f), start = stop - runs_of(len);
      const int per = (len + RUN - 1) / RUN;
      for (; item < end && item < stop; item++) {
        const int section = (int)((item - start) / per),
                  run = (int)(item - start - (int64_t)section * per);
        copy_run(b, section, run, len);
      }
    }
  }
}

__global__ __launch_bounds__(kThreads) void k_page_state(Book k, int32_t *table, int32_t *held,
                                                         int32_t *refs) {
  const size_t n = (size_t)k.sequences * k.slots, step = (size_t)gridDim.x * kThreads;
  const size_t first = (size_t)blockIdx.x * kThreads + threadIdx.x;
  if (table)
    for (size_t i = first; i < n; i += step) table[i] = k.table[i];
  if (held)
    for (size_t i = first; i < (size_t)k.sequences; i += step) held[i] = k.held[i];
  if (refs)
    for (size_t i = first; i < (size_t)k.pages; i += step) refs[i] = k.refs[i];
}

template <int FMT, int HD>
struct GoReserve {
  static void go(const Book &k, const KvView &v, int n, int rows, const int32_t *lens,
                 const int32_t *counts, int32_t *ok, hipStream_t st) {
    // slots of a sequence that the call can touch, up to 64 lanes
    const int most = ((rows - 1) >> k.page_log2) + 2, sections = 2 * v.layers * v.kvh;
    int group = 1;
    while (group < most && group < 64) group *= 2;
    if (most <= group && n * group <= kBook) {
      const int64_t waves = (int64_t)n * sections;
      const unsigned blocks = (unsigned)std::min<int64_t>(256, (waves + kBookWaves - 1) / kBookWaves);
      hipLaunchKernelGGL((k_reserve<FMT, HD>), dim3(blocks), dim3(kBook), 0, st, k, v, n, rows, lens,
                         counts, ok, group);
      return;
    }
    hipLaunchKernelGGL(k_reserve_many, dim3(1), dim3(kBook), 0, st, k, n, rows, lens, counts, ok,
                       group);
    const int each = kThreads / 64;
    hipLaunchKernelGGL((k_copy_tails<FMT, HD>), dim3(n, (sections + each - 1) / each),
                       dim3(kThreads), 0, st, v, k, lens);
  }
};
template <int FMT, int HD>
struct GoCopy {
  static void go(const KvView &to, const KvView &from, const int32_t *sources, int src_sequences,
                 unsigned blocks, hipStream_t st) {
    hipLaunchKernelGGL((k_copy<FMT, HD>), dim3(blocks), dim3(kThreads), 0, st, to, from, sources,
                       src_sequences);
  }
};

void check_pages(const q3h_cache *c, int sequences, const char *who) {
  if (!c) require(false, Q3H_E_ARG, std::string(who) + ": NULL cache");
  if (c->pages <= 0) require(false, Q3H_E_ARG, std::string(who) + ": not a cache of pages");
  if (sequences < 0 || sequences > c->cfg.sequences)
    require(false, Q3H_E_ARG,
            std::string(who) + ": " + std::to_string(sequences) + " sequences of a cache of " +
                std::to_string(c->cfg.sequences));
}

}  // namespace

}  // namespace q3h

using namespace q3h;

extern "C" int q3h_cache_create_paged(q3h_device *dev, const q3h_paged_config *cfg,
                                      q3h_cache **out) {
  return guard([&] {
    require(dev && cfg && out, Q3H_E_ARG, "q3h_cache_create_paged: NULL argument");
    *out = nullptr;
    const q3h_cache_config &f = cfg->cache;
    check_cache_config(f, "q3h_cache_create_paged");
    int log2 = 0;
    for (const int p : {32, 64, 128, 256})
      if (cfg->page_positions == p) log2 = __builtin_ctz(p);
    require(log2 > 0, Q3H_E_ARG,
            "q3h_cache_create_paged: page_positions must be 32, 64, 128 or 256");
    require(cfg->pages > 0 && cfg->pages <= Q3H_MAX_PAGES, Q3H_E_ARG,
            "q3h_cache_create_paged: pages must be in [1, 2^20]");
    const int64_t slots = ((int64_t)f.max_positions + cfg->page_positions - 1) >> log2;
    require(slots * f.sequences <= (1 << 24), Q3H_E_ARG,
            "q3h_cache_create_paged: more than 2^24 pages of all sequences together");
    DeviceScope scope(dev->ordinal);
    q3h_cache *c = new q3h_cache();
    try {
      c->dev = dev;
      c->cfg = f;
      c->pages = cfg->pages;
      c->page_log2 = log2;
      c->slots = (int)slots;
      const size_t need = kv_bytes(f.format, f.layers, f.kv_heads, cfg->page_positions, f.head_dim);
      c->seq_bytes = (need + 255) & ~(size_t)255;
      const size_t all = c->seq_bytes * cfg->pages;
      const size_t words = book_words(f.sequences, c->slots, c->pages);
      c->data = (char *)dev_alloc(all);
      c->state = (int32_t *)dev_alloc(words * sizeof(int32_t));
      check_hip(hipMemset(c->data, 0, all), "zero pages");
      hipLaunchKernelGGL(k_book_clear, dim3(1024), dim3(kThreads), 0, nullptr, book_of(c));
      check_hip(hipGetLastError(), "page table kernel");
      check_hip(hipStreamSynchronize(nullptr), "zero pages sync");
      c->bytes = (int64_t)(all + words * sizeof(int32_t));
    } catch (...) {
      dev_free(c->data);
      dev_free(c->state);
      delete c;
      throw;
    }
    dev->bytes += c->bytes;
    dev->stacks++;
    *out = c;
  });
}

extern "C" int q3h_cache_reserve(q3h_cache *c, int sequences, int rows, const int32_t *lens,
                                 const int32_t *counts, int32_t *ok, void *stream) {
  return guard([&] {
    check_pages(c, sequences, "q3h_cache_reserve");
    require(rows >= 0, Q3H_E_ARG, "q3h_cache_reserve: rows below 0");
    require(rows <= c->cfg.max_positions, Q3H_E_CAPACITY,
            "q3h_cache_reserve: more rows than the cache has positions");
    if (sequences == 0) return;
    require(lens != nullptr, Q3H_E_ARG, "q3h_cache_reserve: NULL lens");
    DeviceScope scope(c->dev->ordinal);
    by_format<GoReserve>(c->cfg.head_dim, c->cfg.format, book_of(c),
                         kv_view(c, 0, sequences, rows, lens, counts), sequences, rows, lens, counts,
                         ok, (hipStream_t)stream);
    check_hip(hipGetLastError(), "cache reserve kernels");
  });
}

extern "C" int q3h_cache_fork(q3h_cache *c, int sequences, const int32_t *sources,
                              const int32_t *lens, void *stream) {
  return guard([&] {
    check_pages(c, sequences, "q3h_cache_fork");
    if (sequences == 0) return;
    require(sources && lens, Q3H_E_ARG, "q3h_cache_fork: NULL sources or lens");
    DeviceScope scope(c->dev->ordinal);
    const Book k = book_of(c);
    hipStream_t st = (hipStream_t)stream;
    if (sequences <= kBook && (int64_t)sequences * c->slots <= kForkSlots) {
      hipLaunchKernelGGL(k_fork_few, dim3(1), dim3(kBook), 0, st, k, sequences, sources, lens);
    } else {
      hipLaunchKernelGGL(k_fork, dim3(sequences), dim3(kThreads), 0, st, k, sources, lens);
      hipLaunchKernelGGL(k_fork_end, dim3(sequences), dim3(kThreads), 0, st, k);
    }
    check_hip(hipGetLastError(), "cache fork kernels");
  });
}

extern "C" int q3h_cache_release(q3h_cache *c, int sequences, const int32_t *lens, void *stream) {
  return guard([&] {
    check_pages(c, sequences, "q3h_cache_release");
    if (sequences == 0) return;
    require(lens != nullptr, Q3H_E_ARG, "q3h_cache_release: NULL lens");
    DeviceScope scope(c->dev->ordinal);
    hipLaunchKernelGGL(k_release, dim3(sequences), dim3(64), 0, (hipStream_t)stream, book_of(c),
                       lens);
    check_hip(hipGetLastError(), "cache release kernel");
  });
}

extern "C" int q3h_cache_compact(q3h_cache *c, int32_t *used, void *stream) {
  return guard([&] {
    check_pages(c, 0, "q3h_cache_compact");
    DeviceScope scope(c->dev->ordinal);
    const Book k = book_of(c);
    hipStream_t st = (hipStream_t)stream;
    const int64_t bytes = (int64_t)c->seq_bytes;
    if (c->pages <= kScan) {
      // (half of the pages at most move)
      const int64_t most = c->pages / 2 * bytes / (64 * kBook);
      const unsigned blocks = (unsigned)std::min<int64_t>(512, std::max<int64_t>(1, most));
      hipLaunchKernelGGL(k_compact, dim3(blocks), dim3(kBook), 0, st, k, c->data, bytes, used);
    } else {
      hipLaunchKernelGGL(k_compact_many, dim3(1), dim3(kBook), 0, st, k, used);
      hipLaunchKernelGGL(k_move, dim3(2048), dim3(kThreads), 0, st, k, c->data, bytes);
    }
    check_hip(hipGetLastError(), "cache compact kernels");
  });
}

extern "C" int q3h_cache_copy(q3h_cache *c, const q3h_cache *src, int sequences,
                              const int32_t *sources, const int32_t *lens, void *stream) {
  return guard([&] {
    require(c && src, Q3H_E_ARG, "q3h_cache_copy: NULL cache");
    require(c != src, Q3H_E_ARG, "q3h_cache_copy: a cache into itself");
    if (sequences < 0 || sequences > c->cfg.sequences)
      require(false, Q3H_E_ARG,
              "q3h_cache_copy: " + std::to_string(sequences) + " sequences of a cache of " +
                  std::to_string(c->cfg.sequences));
    const q3h_cache_config &f = c->cfg, &g = src->cfg;
    require(c->dev->ordinal == src->dev->ordinal, Q3H_E_ARG,
            "q3h_cache_copy: caches of two devices");
    require(f.format == g.format && f.layers == g.layers && f.kv_heads == g.kv_heads &&
                f.head_dim == g.head_dim,
            Q3H_E_ARG, "q3h_cache_copy: caches of other formats, layers, heads or head_dim");
    if (sequences == 0) return;
    require(sources && lens, Q3H_E_ARG, "q3h_cache_copy: NULL sources or lens");
    DeviceScope scope(c->dev->ordinal);
    const KvView to = kv_view(c, 0, sequences, 0, lens, nullptr),
                 from = kv_view(src, 0, src->cfg.sequences, 0, lens, nullptr);
    by_format<GoCopy>(f.head_dim, f.format, to, from, sources, src->cfg.sequences, 2048u,
                      (hipStream_t)stream);
    check_hip(hipGetLastError(), "cache copy kernel");
  });
}

extern "C" int q3h_cache_page_state(const q3h_cache *c, int32_t *table, int32_t *counts,
                                    int32_t *refs, void *stream) {
  return guard([&] {
    check_pages(c, 0, "q3h_cache_page_state");
    if (!table && !counts && !refs) return;
    DeviceScope scope(c->dev->ordinal);
    const Book k = book_of(c);
    const int64_t n = std::max<int64_t>((int64_t)k.sequences * k.slots, k.pages);
    hipLaunchKernelGGL(k_page_state, dim3((unsigned)std::min<int64_t>(256, (n + 255) / 256)),
                       dim3(kThreads), 0, (hipStream_t)stream, k, table, counts, refs);
    check_hip(hipGetLastError(), "cache page state kernel");
  });
}
