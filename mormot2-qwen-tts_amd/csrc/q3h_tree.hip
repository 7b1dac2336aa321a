// q3h_tree.hip - attention of drafted rows over a K/V cache: each row sees the
// positions before the draft and its own path among the drafted rows.
#include <hip/hip_runtime.h>

#include "q3h_draft.h"
#include "q3h_wave.h"

namespace q3h {

namespace {

constexpr int kThreads = 256;

template <int FMT, int HD>
__device__ __forceinline__ float kv_value(const KvView &kv, const KvSeq &s, int64_t at, int e) {
  if constexpr (FMT == Q3H_KV_Q8)
    return (float)reinterpret_cast<const int8_t *>(s.k0)[at * HD + e] * kv_scales(kv, s, HD)[at];
  else if constexpr (FMT == Q3H_KV_F16)
    return (float)reinterpret_cast<const _Float16 *>(s.k0)[at * HD + e];
  else
    return reinterpret_cast<const float *>(s.k0)[at * HD + e];
}

// One workgroup per (query head, row, sequence): a position a thread for the
// scores, an element a thread for the values, with the softmax's running
// maximum and sum over blocks of 256 positions.
template <int FMT, int HD>
__global__ __launch_bounds__(kThreads) void k_attend(AttendRows a) {
  __shared__ float q[HD], p[kThreads], red[kThreads / 64], o[kThreads];
  const int h = blockIdx.y, t = blockIdx.x, b = blockIdx.z, tid = threadIdx.x;
  const KvSeq s = kv_sequence(a.kv, b);
  if (t >= s.count) return;
  const size_t row = (size_t)b * a.kv.rows + t;
  const int g = h / (a.heads / a.kv.kvh);
  uint64_t path = 0;
  bool bad = s.len < 0 || s.len > a.max_len || s.len > s.max_pos - s.count;
  if (a.parents) {
    const Path x = tree_path(a.parents + (size_t)b * a.kv.rows, a.kv.rows);
    path = __shfl(x.rows, t);
    bad = bad || __shfl((int)x.bad, t) != 0;
  }
  float *out = a.out + row * a.ld_out + (size_t)h * HD;
  if (bad) {
    if (tid < HD) out[tid] = NAN;
    return;
  }
  if (tid < HD) q[tid] = a.q[row * a.ldq + (size_t)h * HD + tid] * a.scale;
  __syncthreads();
  const int end = s.len + t + 1;  // (a path's rows are below its own)
  constexpr int PARTS = kThreads / HD;
  const int e = tid % HD, half = tid / HD;
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int j0 = 0; j0 < end; j0 += kThreads) {
    const int j = j0 + tid;
    const bool sees = j < end && (j < s.len || !a.parents || (path >> (j - s.len) & 1));
    float x = -INFINITY;
    if (sees) {
      const int64_t at = kv_row(a.kv, s, 0, g, j);
      x = 0.f;
      for (int i = 0; i < HD; i++) x = fmaf(q[i], kv_value<FMT, HD>(a.kv, s, at, i), x);
    }
    const float wm = wave_max_dpp(x);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = wm;
    __syncthreads();
    float mn = m;
    for (int i = 0; i < kThreads / 64; i++) mn = fmaxf(mn, red[i]);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float f = expf(m - base);
    const float w = sees ? expf(x - base) : 0.f;
    p[tid] = sees ? w : -1.f;  // (negative: not seen)
    const float ws = wave_sum_dpp(w);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = ws;
    __syncthreads();
    l *= f;
    for (int i = 0; i < kThreads / 64; i++) l += red[i];
    acc *= f;
    m = mn;
    for (int i = half; i < kThreads && j0 + i < end; i += PARTS)
      if (!(p[i] < 0.f))
        acc = fmaf(p[i], kv_value<FMT, HD>(a.kv, s, kv_row(a.kv, s, 1, g, j0 + i), e), acc);
  }
  o[tid] = acc;
  __syncthreads();
  if (tid < HD) {
    for (int i = 1; i < PARTS; i++) acc += o[i * HD + tid];
    out[tid] = acc / l;
  }
}

template <int HD>
void launch(const AttendRows &a, int fmt, hipStream_t st) {
  const dim3 grid(a.kv.rows, a.heads, a.kv.sequences);
  if (fmt == Q3H_KV_F32)
    hipLaunchKernelGGL((k_attend<Q3H_KV_F32, HD>), grid, dim3(kThreads), 0, st, a);
  else if (fmt == Q3H_KV_F16)
    hipLaunchKernelGGL((k_attend<Q3H_KV_F16, HD>), grid, dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((k_attend<Q3H_KV_Q8, HD>), grid, dim3(kThreads), 0, st, a);
}

}  // namespace

size_t attend_part_bytes(int, int, int, int, int, int) { return 0; }

void launch_cache_attend(const AttendRows &a, int hd, int fmt, hipStream_t st) {
  if (hd == 64)
    launch<64>(a, fmt, st);
  else
    launch<128>(a, fmt, st);
}

}  // namespace q3h
