// Verification of drafted tokens against the target's probabilities, from
// given random numbers: what follows the MTP-verify attention and the model's
// head in a step.  No counterpart in the reference (its engine samples).
//
// Sequence b holds n_b <= K drafts x_0 .. x_{n_b - 1}, the target's
// probabilities p_i of position i (K + 1 rows of V) and, unless its drafts
// were chosen outright, the draft model's q_i.
//   Draft i is accepted iff u_i * q_i(x_i) < p_i(x_i) (q_i(x_i) = 1 for drafts
//   chosen outright); a is the number accepted before the first refusal.
//   w = max(p_a - q_a, 0) where draft a was refused (p_a with x_a taken out
//   for drafts chosen outright), p_a where all were accepted; where that
//   leaves no weight (a refusal that only rounding explains), w = p_a.
//   The new token is the lowest v with w_0 + .. + w_v > s * sum(w).
// So the output tokens are distributed as the target's own samples.
//
// Bound by memory: one row of p and one of q per sequence, 2 V elements; the
// acceptance tests read 2 K elements.  The products of the tests, the weights
// and their sums are formed in float64 (products of two 24-bit values are
// exact there), so a decision differs from the real numbers' only within
// 2^-50 or so of a border, and nothing depends on the launch shape's order:
// each sum has a fixed order.
//
// Two launches.  The first spreads the rows over the chip: one wave sums one
// piece of kPiece weights, 16 a lane, and writes the sum; where a refusal leaves
// the piece no weight, that of p alone too.  The second takes one work-group per
// sequence, finds the piece the sample falls in from the V / kPiece sums, rereads
// that piece alone (it is still in cache) and finds the token; where the weights'
// sums are all zero it does so once more with p's, so a row without weight costs a
// search and not a pass.
//
// Loads: an fp32 wave has its p and q, eight 16-byte loads a lane, in flight
// together (256 x 4 over 152,000: 5.9 TB/s, 52.7 us on rows not in cache).  A 16-bit
// one converts inside the branch of each load and so waits for its four one by one;
// many waves hide that (the same call in bf16: 4.9 TB/s, 31.9 us), few do not (48 x 6
// over 65,537: the first launch takes 6.4 us where a launch alone takes 3.7).
#include "k8v4_common.h"

namespace k8v4 {
namespace {

constexpr int kPiece = 1024;           // elements of one partial sum
constexpr int kPerLane = kPiece / 64;  // 16 in the first kernel
constexpr int kScanWaves = 4;          // pieces of one work-group of the first kernel
constexpr int kMaxDrafts = 63;         // one lane per draft, and one row more

struct VerifyArgs {
  const void *target;
  int64_t t_seq, t_row;  // elements between sequences / positions
  const void *draft;     // nullable
  int64_t d_seq, d_row;
  const void *tokens;  // int32 or int64 [batch][K]
  int tokens64;
  int64_t tok_stride;
  const int32_t *counts;  // nullable: K
  const float *accept_u;
  int64_t u_stride;
  const float *sample_u;
  const int32_t *seq_lens;  // nullable
  int64_t *out_tokens;
  int64_t out_stride;
  int32_t *accepted;
  int32_t *next_lens;  // nullable
  double *sums;        // [batch][2][pieces]: of the weights, and of p alone (see verify_sum_kernel)
  int32_t *chain;      // [batch]: accepted drafts
  int batch, drafts, vocab, pieces;
};

template <typename T>
__device__ __forceinline__ float to_float(T x) {
  return static_cast<float>(x);
}

__device__ __forceinline__ int64_t token_at(const VerifyArgs &a, int b, int i) {
  const int64_t at = b * a.tok_stride + i;
  return a.tokens64 ? static_cast<const int64_t *>(a.tokens)[at]
                    : static_cast<int64_t>(static_cast<const int32_t *>(a.tokens)[at]);
}

__device__ __forceinline__ int draft_count(const VerifyArgs &a, int b) {
  const int n = a.counts ? a.counts[b] : a.drafts;
  return min(max(n, 0), a.drafts);
}

// Drafts of sequence b accepted before the first refusal (the same in every
// lane): lane i tests draft i.  A token outside the vocabulary is refused.
template <typename T>
__device__ int accept_chain(const VerifyArgs &a, int b, int n, int lane) {
  bool ok = false;
  if (lane < n) {
    const int64_t x = token_at(a, b, lane);
    if (x >= 0 && x < a.vocab) {
      const double p = to_float(static_cast<const T *>(a.target)[b * a.t_seq + lane * a.t_row + x]);
      const double q = a.draft ? to_float(static_cast<const T *>(a.draft)[b * a.d_seq + lane * a.d_row + x]) : 1.f;
      ok = static_cast<double>(a.accept_u[b * a.u_stride + lane]) * q < p;
    }
  }
  return min(__builtin_ctzll(~__ballot(ok)), n);  // lane 63 never tests a draft
}

// The weight of one element: p - q where positive (a NaN has none).
__device__ __forceinline__ double weight(float p, float q) {
  const double w = static_cast<double>(p) - static_cast<double>(q);
  return w > 0.0 ? w : 0.0;
}

// Where the weights of sequence b come from, once its chain is known.
template <typename T>
struct Weights {
  const T *p;
  const T *q;   // nullable
  int64_t out;  // element taken out (-1: none)
};
template <typename T>
__device__ __forceinline__ Weights<T> weights_of(const VerifyArgs &a, int b, int n, int acc) {
  Weights<T> w;
  w.p = static_cast<const T *>(a.target) + b * a.t_seq + acc * a.t_row;
  w.q = nullptr;
  w.out = -1;
  if (acc < n) {
    if (a.draft)
      w.q = static_cast<const T *>(a.draft) + b * a.d_seq + acc * a.d_row;
    else
      w.out = token_at(a, b, acc);
  }
  return w;
}

// N consecutive elements from `at` on (those from `vocab` on read as 0).  One
// wide load where all of them exist; rows of an odd vocabulary start at any
// element, which the memory system takes.
template <typename T, int N>
__device__ __forceinline__ void load_run(const T *row, int64_t at, int vocab, float (&x)[N]) {
  if (at + N <= vocab) {
    T raw[N];
    __builtin_memcpy(raw, row + at, sizeof(raw));
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_float(raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = at + i < vocab ? to_float(row[at + i]) : 0.f;
  }
}

__device__ __forceinline__ double wave_sum_f64(double x) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) x += __shfl_xor(x, m, kWave);
  return x;
}

template <typename T>
__global__ __launch_bounds__(64 * kScanWaves) void verify_sum_kernel(VerifyArgs a) {
  constexpr int VEC = 16 / sizeof(T);  // elements of one 16-byte load
  constexpr int STEPS = kPerLane / VEC;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = threadIdx.x / kWave;
  const int b = blockIdx.y;
  const int piece = static_cast<int>(blockIdx.x) * kScanWaves + wave;
  if (piece >= a.pieces) return;
  const int n = draft_count(a, b);
  const int acc = accept_chain<T>(a, b, n, lane);
  const Weights<T> w = weights_of<T>(a, b, n, acc);
  if (piece == 0 && lane == 0) a.chain[b] = acc;
  float p[STEPS][VEC], q[STEPS][VEC] = {};
  const int64_t at0 = static_cast<int64_t>(piece) * kPiece + lane * VEC;
#pragma unroll
  for (int s = 0; s < STEPS; ++s) load_run<T, VEC>(w.p, at0 + s * kWave * VEC, a.vocab, p[s]);
  if (w.q) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) load_run<T, VEC>(w.q, at0 + s * kWave * VEC, a.vocab, q[s]);
  }
  double *sums = a.sums + static_cast<int64_t>(b) * 2 * a.pieces + piece;
  double sum = 0.0;
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const double x = weight(p[s][i], q[s][i]);
      sum += at0 + s * kWave * VEC + i == w.out ? 0.0 : x;
    }
  sum = wave_sum_f64(sum);
  if (lane == 0) sums[0] = sum;
  if (acc < n && !(sum > 0.0)) {
    // Read by the second launch only if no piece has any weight left.
    sum = 0.0;
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += weight(p[s][i], 0.f);
    sum = wave_sum_f64(sum);
    if (lane == 0) sums[a.pieces] = sum;
  }
}

constexpr int kPickThreads = 256;
constexpr int kPickWaves = kPickThreads / kWave;

// Inclusive scan over the work-group; `total` is the whole sum.  Every thread
// calls it.
__device__ double block_scan(double x, double *lds, double *total) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    const double y = __shfl_up(x, m, kWave);
    if (lane >= m) x += y;
  }
  __syncthreads();  // the previous scan's words have been read
  if (lane == kWave - 1) lds[wave] = x;
  __syncthreads();
  double before = 0.0, all = 0.0;
#pragma unroll
  for (int v = 0; v < kPickWaves; ++v) {
    if (v < wave) before += lds[v];
    all += lds[v];
  }
  *total = all;
  return before + x;
}

// The lowest (or highest) of the work-group's candidates; INT_MAX (-1) if none.
__device__ int block_min(int x, int *lds) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) x = min(x, __shfl_xor(x, m, kWave));
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = x;
  __syncthreads();
  int r = lds[0];
#pragma unroll
  for (int v = 1; v < kPickWaves; ++v) r = min(r, lds[v]);
  return r;
}
__device__ int block_max(int x, int *lds) { return -block_min(-x, lds); }

struct PickShared {
  double scan[kPickWaves];
  int red[kPickWaves];
  double base;  // weight before the chosen piece
};

// The lowest element of [at, at + kPiece) whose running weight, `base` before
// it, passes `target`; where rounding lets none pass, the last one with any
// weight (-1: none has).
template <typename T>
__device__ int pick_in_piece(const VerifyArgs &a, const Weights<T> &w, int64_t at, double base, double target,
                             PickShared *sh) {
  constexpr int EL = kPiece / kPickThreads;
  float p[EL], q[EL] = {};
  const int64_t at0 = at + static_cast<int64_t>(threadIdx.x) * EL;
  load_run<T, EL>(w.p, at0, a.vocab, p);
  if (w.q) load_run<T, EL>(w.q, at0, a.vocab, q);
  double x[EL], sum = 0.0;
#pragma unroll
  for (int i = 0; i < EL; ++i) {
    x[i] = at0 + i == w.out ? 0.0 : weight(p[i], q[i]);
    sum += x[i];
  }
  double total;
  double run = base + (block_scan(sum, sh->scan, &total) - sum);
  int first = INT32_MAX, last = -1;
#pragma unroll
  for (int i = 0; i < EL; ++i) {
    run += x[i];
    if (x[i] > 0.0) {
      if (run > target && first == INT32_MAX) first = static_cast<int>(at0 + i);
      last = static_cast<int>(at0 + i);
    }
  }
  first = block_min(first, sh->red);
  if (first != INT32_MAX) return first;
  return block_max(last, sh->red);
}

// The sampled token from the per-piece sums, or -1 where no element weighs anything.
template <typename T>
__device__ int pick(const VerifyArgs &a, const Weights<T> &w, float u, PickShared *sh, const double *sums) {
  // Thread t holds the consecutive pieces t * per .. t * per + per - 1.
  const int per = (a.pieces + kPickThreads - 1) / kPickThreads;
  const int p0 = static_cast<int>(threadIdx.x) * per, p1 = min(p0 + per, a.pieces);
  double mine = 0.0;
  for (int i = p0; i < p1; ++i) mine += sums[i];
  double total;
  const double before = block_scan(mine, sh->scan, &total) - mine;
  if (!(total > 0.0)) return -1;
  const double target = static_cast<double>(u) * total;
  int first = INT32_MAX, last = -1;
  double run = before;
  for (int i = p0; i < p1; ++i) {
    const double x = sums[i];
    run += x;
    if (x > 0.0) {
      if (run > target && first == INT32_MAX) first = i;
      last = i;
    }
  }
  int chosen = block_min(first, sh->red);
  if (chosen == INT32_MAX) chosen = block_max(last, sh->red);
  if (chosen >= p0 && chosen < p1) {
    double base = before;
    for (int i = p0; i < chosen; ++i) base += sums[i];
    sh->base = base;
  }
  __syncthreads();
  return pick_in_piece(a, w, static_cast<int64_t>(chosen) * kPiece, sh->base, target, sh);
}

template <typename T>
__global__ __launch_bounds__(kPickThreads) void verify_pick_kernel(VerifyArgs a) {
  __shared__ PickShared sh;
  const int b = blockIdx.x;
  const int n = draft_count(a, b);
  const int acc = a.chain[b];
  const float u = a.sample_u[b];
  const double *sums = a.sums + static_cast<int64_t>(b) * 2 * a.pieces;
  Weights<T> w = weights_of<T>(a, b, n, acc);
  int token = pick<T>(a, w, u, &sh, sums);
  if (token < 0 && acc < n) {
    // Refused, and nothing is left of the row: the target's own probabilities.
    w.q = nullptr;
    w.out = -1;
    token = pick<T>(a, w, u, &sh, sums + a.pieces);
  }
  for (int j = threadIdx.x; j <= a.drafts; j += kPickThreads)
    a.out_tokens[b * a.out_stride + j] = j < acc ? token_at(a, b, j) : j == acc ? token : -1;
  if (threadIdx.x == 0) {
    a.accepted[b] = acc;
    if (a.next_lens) a.next_lens[b] = a.seq_lens[b] + acc + 1;
  }
}

template <typename T>
void launch(const VerifyArgs &a, hipStream_t s) {
  const unsigned groups = static_cast<unsigned>((a.pieces + kScanWaves - 1) / kScanWaves);
  verify_sum_kernel<T><<<dim3(groups, static_cast<unsigned>(a.batch)), dim3(64 * kScanWaves), 0, s>>>(a);
  verify_pick_kernel<T><<<dim3(static_cast<unsigned>(a.batch)), dim3(kPickThreads), 0, s>>>(a);
}

constexpr int64_t kMaxBatch = 65535;  // the first launch's second grid dimension
constexpr int64_t kMaxVocab = int64_t(1) << 24;

int64_t chain_bytes(int64_t batch) { return (batch * 4 + 255) / 256 * 256; }

}  // namespace
}  // namespace k8v4

extern "C" int64_t k8v4_verify_drafts_workspace_bytes(int64_t batch, int64_t vocab) {
  using namespace k8v4;
  if (batch < 0 || batch > kMaxBatch || vocab < 1 || vocab > kMaxVocab) return -1;
  return chain_bytes(batch) + batch * 2 * ((vocab + kPiece - 1) / kPiece) * 8;
}

extern "C" int k8v4_verify_drafts(const void *target_probs, int dtype, int64_t target_seq_stride,
                                  int64_t target_row_stride, const void *draft_probs, int64_t draft_seq_stride,
                                  int64_t draft_row_stride, const void *draft_tokens, int tokens_are_int64,
                                  int64_t token_stride, const int32_t *num_drafts, const float *accept_uniform,
                                  int64_t uniform_stride, const float *sample_uniform, const int32_t *seq_lens,
                                  int64_t batch, int max_drafts, int64_t vocab, int64_t *out_tokens,
                                  int64_t out_stride, int32_t *accepted, int32_t *next_lens, void *workspace,
                                  int64_t workspace_bytes, void *stream) {
  using namespace k8v4;
  clear_error();
  K8V4_REQUIRE(dtype == K8V4_F16 || dtype == K8V4_BF16 || dtype == K8V4_F32,
               "probabilities must be fp16, bf16 or fp32");
  K8V4_REQUIRE(batch >= 0 && batch <= kMaxBatch, "batch must be 0 .. %lld", static_cast<long long>(kMaxBatch));
  K8V4_REQUIRE(max_drafts >= 0 && max_drafts <= kMaxDrafts, "0 to %d drafts a sequence, got %d", kMaxDrafts, max_drafts);
  K8V4_REQUIRE(vocab >= 1 && vocab <= kMaxVocab, "vocabulary must be 1 .. %lld", static_cast<long long>(kMaxVocab));
  if (batch == 0) return K8V4_OK;
  K8V4_REQUIRE(target_probs && sample_uniform && out_tokens && accepted && workspace &&
                   (max_drafts == 0 || (draft_tokens && accept_uniform)),
               "null pointer");
  K8V4_REQUIRE(!next_lens || seq_lens, "next_lens needs seq_lens");
  K8V4_REQUIRE(target_row_stride >= vocab || max_drafts == 0, "target row stride shorter than the vocabulary");
  K8V4_REQUIRE(target_seq_stride >= vocab || batch == 1, "target sequence stride shorter than the vocabulary");
  if (draft_probs && max_drafts) {
    K8V4_REQUIRE(draft_row_stride >= vocab || max_drafts == 1, "draft row stride shorter than the vocabulary");
    K8V4_REQUIRE(draft_seq_stride >= vocab || batch == 1, "draft sequence stride shorter than the vocabulary");
  }
  K8V4_REQUIRE(out_stride > max_drafts || batch == 1, "out_tokens row stride shorter than drafts + 1");
  K8V4_REQUIRE(token_stride >= max_drafts || batch == 1, "draft_tokens row stride shorter than the drafts");
  K8V4_REQUIRE(uniform_stride >= max_drafts || batch == 1, "accept_uniform row stride shorter than the drafts");
  const int esize = dtype == K8V4_F32 ? 4 : 2;
  const auto misaligned = [](const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
  K8V4_REQUIRE(!misaligned(target_probs, esize) && !misaligned(draft_probs, esize) && !misaligned(out_tokens, 8) &&
                   !misaligned(draft_tokens, tokens_are_int64 ? 8 : 4) && !misaligned(accept_uniform, 4) &&
                   !misaligned(sample_uniform, 4) && !misaligned(num_drafts, 4) && !misaligned(seq_lens, 4) &&
                   !misaligned(accepted, 4) && !misaligned(next_lens, 4),
               "misaligned pointer");
  K8V4_REQUIRE(!misaligned(workspace, 16), "workspace must be 16-byte aligned");
  const int64_t need = k8v4_verify_drafts_workspace_bytes(batch, vocab);
  if (workspace_bytes < need) {
    set_error("verify workspace holds %lld bytes, the batch needs %lld", static_cast<long long>(workspace_bytes),
              static_cast<long long>(need));
    return K8V4_ERR_WORKSPACE;
  }

  VerifyArgs a;
  a.target = target_probs;
  a.t_seq = target_seq_stride;
  a.t_row = target_row_stride;
  a.draft = max_drafts ? draft_probs : nullptr;
  a.d_seq = draft_seq_stride;
  a.d_row = draft_row_stride;
  a.tokens = draft_tokens;
  a.tokens64 = tokens_are_int64 != 0;
  a.tok_stride = token_stride;
  a.counts = num_drafts;
  a.accept_u = accept_uniform;
  a.u_stride = uniform_stride;
  a.sample_u = sample_uniform;
  a.seq_lens = seq_lens;
  a.out_tokens = out_tokens;
  a.out_stride = out_stride;
  a.accepted = accepted;
  a.next_lens = next_lens;
  a.chain = static_cast<int32_t *>(workspace);
  a.sums = reinterpret_cast<double *>(static_cast<char *>(workspace) + chain_bytes(batch));
  a.batch = static_cast<int>(batch);
  a.drafts = max_drafts;
  a.vocab = static_cast<int>(vocab);
  a.pieces = static_cast<int>((vocab + kPiece - 1) / kPiece);
  auto s = static_cast<hipStream_t>(stream);
  if (dtype == K8V4_F32)
    launch<float>(a, s);
  else if (dtype == K8V4_BF16)
    launch<__bf16>(a, s);
  else
    launch<_Float16>(a, s);
  return launch_status("k8v4_verify_drafts");
}
