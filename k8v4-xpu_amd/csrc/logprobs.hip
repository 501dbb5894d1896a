// Log probabilities of given tokens, their ranks, the entropies and the likeliest
// tokens of rows of logits.  No counterpart in the reference (its engine's).
//
// With m the row's largest logit, y_v = x_v - m and S = sum exp(y_v):
//   log p_v = y_v - log S,   H = log S - sum(y_v exp(y_v)) / S.
// The rank of token t is 1 + the number of tokens ahead of it: of larger logit, or
// of equal logit and lower index; the likeliest tokens are those of rank 1, 2, ...
// A logit that is minus infinity or NaN has no probability: its log is minus
// infinity, its rank 0, and it is none of the likeliest.
//
// S is kept as 1 + r with r the sum without one largest element, and log S as
// log1p(r), so that a token of probability near 1 keeps its log to fp32's relative
// accuracy.
#include "k8v4_common.h"

namespace k8v4 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 64;

struct LogprobArgs {
  const void *logits;
  int64_t row_stride;  // elements
  const void *tokens;  // nullable; int32 or int64
  int tokens64;
  int64_t rows;
  int vocab, top;
  float *logprobs;
  int32_t *ranks;
  float *entropy;  // nullable
  int64_t *top_ids;
  int64_t ids_stride;
  float *top_logprobs;
  int64_t lps_stride;
};

template <typename T>
__device__ __forceinline__ float logit(T x) {
  const float f = static_cast<float>(x);
  return f != f ? -INFINITY : f;
}

// Whether (x, i) comes ahead of (y, j).
__device__ __forceinline__ bool ahead(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

struct Shared {
  float x[kThreads / kWave];
  int i[kThreads / kWave];
  double d[kThreads / kWave];
};

// The foremost of the work-group's elements.
__device__ void block_first(float &x, int &i, Shared &sh) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    const float y = __shfl_xor(x, m, kWave);
    const int j = __shfl_xor(i, m, kWave);
    if (ahead(y, j, x, i)) {
      x = y;
      i = j;
    }
  }
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) {
    sh.x[threadIdx.x / kWave] = x;
    sh.i[threadIdx.x / kWave] = i;
  }
  __syncthreads();
  x = sh.x[0];
  i = sh.i[0];
#pragma unroll
  for (int w = 1; w < kThreads / kWave; ++w)
    if (ahead(sh.x[w], sh.i[w], x, i)) {
      x = sh.x[w];
      i = sh.i[w];
    }
}

__device__ double block_sum(double x, Shared &sh) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) x += __shfl_xor(x, m, kWave);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) sh.d[threadIdx.x / kWave] = x;
  __syncthreads();
  double r = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / kWave; ++w) r += sh.d[w];
  return r;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void logprob_kernel(LogprobArgs a) {
  __shared__ Shared sh;
  const int64_t row = blockIdx.x;
  const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
  int64_t t = -1;
  if (a.tokens)
    t = a.tokens64 ? static_cast<const int64_t *>(a.tokens)[row] : static_cast<const int32_t *>(a.tokens)[row];
  const bool inside = t >= 0 && t < a.vocab;
  const float xt = inside ? logit(x[t]) : -INFINITY;
  float m = -INFINITY;
  int im = INT32_MAX;
  int before = 0;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
    const float v = logit(x[i]);
    if (ahead(v, i, m, im)) {
      m = v;
      im = i;
    }
    before += ahead(v, i, xt, static_cast<int>(t));
  }
  block_first(m, im, sh);
  const bool some = m > -INFINITY;
  double rest = 0.0, mean = 0.0;
  for (int i = threadIdx.x; i < a.vocab && some; i += kThreads) {
    const float v = logit(x[i]);
    if (i == im) continue;
    const float y = v == m ? 0.f : v - m, e = expf(y);
    rest += e;
    if (e > 0.f) mean += y * e;
  }
  rest = block_sum(rest, sh);
  mean = block_sum(mean, sh);
  before = static_cast<int>(block_sum(before, sh));
  const float log_s = static_cast<float>(log1p(rest));
  if (threadIdx.x == 0) {
    const bool there = some && xt > -INFINITY;
    if (a.tokens) {
      a.logprobs[row] = there ? (xt == m ? 0.f : xt - m) - log_s : -INFINITY;
      a.ranks[row] = there ? before + 1 : 0;
    }
    if (a.entropy) a.entropy[row] = some ? static_cast<float>(log1p(rest) - mean / (1.0 + rest)) : 0.f;
  }
  float last = INFINITY;
  int ilast = -1;
  for (int k = 0; k < a.top; ++k) {
    float best = -INFINITY;
    int ibest = INT32_MAX;
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
      const float v = logit(x[i]);
      if (ahead(last, ilast, v, i) && ahead(v, i, best, ibest)) {
        best = v;
        ibest = i;
      }
    }
    block_first(best, ibest, sh);
    const bool there = best > -INFINITY;
    if (threadIdx.x == 0) {
      a.top_ids[row * a.ids_stride + k] = there ? ibest : -1;
      a.top_logprobs[row * a.lps_stride + k] = there ? (best == m ? 0.f : best - m) - log_s : -INFINITY;
    }
    last = best;
    ilast = ibest;
  }
}

constexpr int64_t kMaxVocab = int64_t(1) << 24;

}  // namespace
}  // namespace k8v4

extern "C" int64_t k8v4_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int top) {
  using namespace k8v4;
  if (rows < 0 || rows > INT32_MAX || vocab < 1 || vocab > kMaxVocab || top < 0 || top > kMaxTop) return -1;
  return 0;
}

extern "C" int k8v4_token_logprobs(const void *logits, int dtype, int64_t row_stride, const void *tokens,
                                   int tokens_are_int64, int64_t rows, int64_t vocab, int top, float *logprobs,
                                   int32_t *ranks, float *entropy, int64_t *top_ids, int64_t ids_stride,
                                   float *top_logprobs, int64_t lps_stride, void *workspace, int64_t workspace_bytes,
                                   void *stream) {
  using namespace k8v4;
  clear_error();
  K8V4_REQUIRE(dtype == K8V4_F16 || dtype == K8V4_BF16 || dtype == K8V4_F32, "logits must be fp16, bf16 or fp32");
  K8V4_REQUIRE(rows >= 0 && rows <= INT32_MAX, "rows must be 0 .. 2^31 - 1");
  K8V4_REQUIRE(vocab >= 1 && vocab <= kMaxVocab, "vocabulary must be 1 .. %lld", static_cast<long long>(kMaxVocab));
  K8V4_REQUIRE(top >= 0 && top <= kMaxTop, "0 to %d likeliest tokens, got %d", kMaxTop, top);
  if (rows == 0) return K8V4_OK;
  K8V4_REQUIRE(logits && (!tokens || (logprobs && ranks)) && (top == 0 || (top_ids && top_logprobs)), "null pointer");
  K8V4_REQUIRE(row_stride >= vocab || rows == 1, "logits row stride shorter than the vocabulary");
  K8V4_REQUIRE(rows == 1 || (ids_stride >= top && lps_stride >= top), "likeliest tokens' row stride shorter than their count");
  const auto misaligned = [](const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
  K8V4_REQUIRE(!misaligned(logits, dtype == K8V4_F32 ? 4 : 2) && !misaligned(tokens, tokens_are_int64 ? 8 : 4) &&
                   !misaligned(logprobs, 4) && !misaligned(ranks, 4) && !misaligned(entropy, 4) &&
                   !misaligned(top_ids, 8) && !misaligned(top_logprobs, 4),
               "misaligned pointer");
  K8V4_REQUIRE(!misaligned(workspace, 16), "workspace must be 16-byte aligned");
  const int64_t need = k8v4_token_logprobs_workspace_bytes(rows, vocab, top);
  if (workspace_bytes < need || (need && !workspace)) {
    set_error("log probability workspace holds %lld bytes, the rows need %lld", static_cast<long long>(workspace_bytes),
              static_cast<long long>(need));
    return K8V4_ERR_WORKSPACE;
  }
  LogprobArgs a;
  a.logits = logits;
  a.row_stride = row_stride;
  a.tokens = tokens;
  a.tokens64 = tokens_are_int64 != 0;
  a.rows = rows;
  a.vocab = static_cast<int>(vocab);
  a.top = top;
  a.logprobs = logprobs;
  a.ranks = ranks;
  a.entropy = entropy;
  a.top_ids = top_ids;
  a.ids_stride = ids_stride;
  a.top_logprobs = top_logprobs;
  a.lps_stride = lps_stride;
  const dim3 grid(static_cast<unsigned>(rows));
  auto s = static_cast<hipStream_t>(stream);
  if (dtype == K8V4_F32)
    logprob_kernel<float><<<grid, dim3(kThreads), 0, s>>>(a);
  else if (dtype == K8V4_BF16)
    logprob_kernel<__bf16><<<grid, dim3(kThreads), 0, s>>>(a);
  else
    logprob_kernel<_Float16><<<grid, dim3(kThreads), 0, s>>>(a);
  return launch_status("k8v4_token_logprobs");
}
