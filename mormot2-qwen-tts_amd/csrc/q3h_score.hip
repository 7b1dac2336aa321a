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

constexpr int kThreads = 256, kWaves = kThreads / 64;

template <bool BF16>
__device__ __forceinline__ float logit(const void *p, size_t i) {
  if constexpr (BF16)
    return __uint_as_float((uint32_t) static_cast<const uint16_t *>(p)[i] << 16);
  else
    return static_cast<const float *>(p)[i];
}

// whether (x, i) comes before (y, j) from the top: larger first, of equal ones
// the lower token, NaN last (among themselves by token)
__device__ __forceinline__ bool before(float x, int i, float y, int j) {
  const bool nx = x != x, ny = y != y;
  if (nx != ny) return ny;
  if (!nx && x != y) return x > y;
  return i < j;
}

// One workgroup per row: the maximum, then the sums of e^(x - max) and of
// (x - max) e^(x - max), then the top tokens one by one.
template <bool BF16>
__global__ __launch_bounds__(kThreads) void k_score(ScoreRows a) {
  __shared__ float rv[kWaves], rs[kWaves], rt[kWaves];
  __shared__ int ri[kWaves];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const void *x = static_cast<const char *>(a.logits) + (size_t)r * a.ld * (BF16 ? 2 : 4);
  float m = -INFINITY;
  for (int i = tid; i < a.vocab; i += kThreads) m = fmaxf(m, logit<BF16>(x, i));
  m = wave_max_dpp(m);
  if (lane == 0) rv[wave] = m;
  __syncthreads();
  for (int i = 0; i < kWaves; i++) m = fmaxf(m, rv[i]);
  float s = 0.f, u = 0.f;
  for (int i = tid; i < a.vocab; i += kThreads) {
    const float d = logit<BF16>(x, i) - m, e = expf(d);
    s += e;
    if (e != 0.f) u += d * e;
  }
  s = wave_sum_dpp(s);
  u = wave_sum_dpp(u);
  if (lane == 0) {
    rs[wave] = s;
    rt[wave] = u;
  }
  __syncthreads();
  s = u = 0.f;
  for (int i = 0; i < kWaves; i++) {
    s += rs[i];
    u += rt[i];
  }
  const float ls = logf(s);
  for (int i = tid; i < a.tokens_per_row; i += kThreads) {
    const int t = a.tokens[(size_t)r * a.tokens_per_row + i];
    a.logprobs[(size_t)r * a.tokens_per_row + i] =
        t >= 0 && t < a.vocab ? logit<BF16>(x, t) - m - ls : NAN;
  }
  if (tid == 0 && a.entropy) a.entropy[r] = ls - u / s;
  float lv = 0.f;
  int li = -1;
  for (int k = 0; k < a.top_k; k++) {
    float bv = NAN;
    int bi = INT32_MAX;
    for (int i = tid; i < a.vocab; i += kThreads) {
      const float v = logit<BF16>(x, i);
      if ((li < 0 || before(lv, li, v, i)) && before(v, i, bv, bi)) {
        bv = v;
        bi = i;
      }
    }
    for (int o = 32; o > 0; o >>= 1) {
      const float v2 = __shfl_xor(bv, o);
      const int i2 = __shfl_xor(bi, o);
      if (before(v2, i2, bv, bi)) {
        bv = v2;
        bi = i2;
      }
    }
    __syncthreads();
    if (lane == 0) {
      rv[wave] = bv;
      ri[wave] = bi;
    }
    __syncthreads();
    lv = rv[0];
    li = ri[0];
    for (int i = 1; i < kWaves; i++)
      if (before(rv[i], ri[i], lv, li)) {
        lv = rv[i];
        li = ri[i];
      }
    if (tid == 0) {
      a.top_ids[(size_t)r * a.top_k + k] = li;
      a.top_logprobs[(size_t)r * a.top_k + k] = lv - m - ls;
    }
  }
}

}  // namespace

size_t score_work_bytes(int, int, int) { return 0; }

void launch_token_scores(const ScoreRows &a, hipStream_t st) {
  if (a.bf16)
    hipLaunchKernelGGL(k_score<true>, dim3(a.rows), dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL(k_score<false>, dim3(a.rows), dim3(kThreads), 0, st, a);
}

}  // namespace q3h

using namespace q3h;

extern "C" int64_t q3h_token_logprobs_workspace(int rows, int vocab, int top_k) {
  int64_t bytes = 0;
  const int rc = guard([&] {
    require(rows >= 0 && vocab > 0 && top_k >= 0 && top_k <= Q3H_TOP_MAX && top_k <= vocab,
            Q3H_E_ARG, "q3h_token_logprobs_workspace: invalid argument");
    if (rows > 0) bytes = (int64_t)score_work_bytes(rows, vocab, top_k);
  });
  return rc ? rc : bytes;
}

extern "C" int q3h_token_logprobs(q3h_device *dev, const q3h_score_args *p, void *stream) {
  return guard([&] {
    require(dev && p, Q3H_E_ARG, "q3h_token_logprobs: NULL argument");
    require(p->rows >= 0 && p->vocab > 0 && p->vocab <= (1 << 30), Q3H_E_ARG,
            "q3h_token_logprobs: bad rows or vocab");
    require(p->dtype == Q3H_F32 || p->dtype == Q3H_BF16, Q3H_E_ARG,
            "q3h_token_logprobs: dtype must be Q3H_F32 or Q3H_BF16");
    require(p->tokens_per_row >= 0, Q3H_E_ARG, "q3h_token_logprobs: negative tokens_per_row");
    require(p->top_k >= 0 && p->top_k <= Q3H_TOP_MAX && p->top_k <= p->vocab, Q3H_E_ARG,
            "q3h_token_logprobs: top_k must be in [0, min(vocab, " + std::to_string(Q3H_TOP_MAX) +
                ")]");
    if (p->rows == 0) return;
    require(p->logits != nullptr, Q3H_E_ARG, "q3h_token_logprobs: NULL logits");
    require(p->ld >= p->vocab, Q3H_E_ARG, "q3h_token_logprobs: rows overlap (ld below vocab)");
    require(p->tokens_per_row == 0 || (p->tokens && p->logprobs), Q3H_E_ARG,
            "q3h_token_logprobs: NULL tokens or logprobs");
    require(p->top_k == 0 || (p->top_ids && p->top_logprobs), Q3H_E_ARG,
            "q3h_token_logprobs: NULL top_ids or top_logprobs");
    const size_t need = score_work_bytes(p->rows, p->vocab, p->top_k);
    require(need == 0 || (p->workspace && p->workspace_bytes >= (int64_t)need &&
                          (uintptr_t)p->workspace % 256 == 0),
            Q3H_E_ARG, "q3h_token_logprobs: a workspace of " + std::to_string(need) +
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
