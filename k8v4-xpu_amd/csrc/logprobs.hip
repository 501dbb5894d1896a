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
//
// One pass.  A wave keeps one running maximum; a batch of elements below it, which
// most are, takes one fma, one clamp (for NaN and minus infinity), one exponential and
// two additions an element, a comparison with the given token (counted in scalars) and
// half an instruction of a maximum; a batch with a new maximum rescales the sums.  The
// maxima of 128-byte chunks go to the LDS; the K foremost chunks hold the K likeliest
// tokens, which are read again and ranked.  Few rows are cut into slices and joined by
// a second launch.
//
// Bound by memory, closely followed by issue (12 slots an element): 2048 x 152000 bf16
// with 20 tokens a row 145 us, 4.3 TB/s (a sum over 2 GiB reads 4.0); calls of a few
// rows by latency, two launches of about 7 and 5 us.
#include "k8v4_common.h"

namespace k8v4 {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxTop = 64;
constexpr int kMaxSlices = 64;  // one lane each when they are joined
constexpr int kGroupLanes = 8;  // lanes whose vectors make a chunk
constexpr int kStream = 4;      // vectors of a thread in flight
constexpr int kMaxListed = 256;
constexpr int kSliceUnit = 2048;        // elements of a slice at least, and its length's unit
constexpr int kMaxSliceLen = 1 << 18;   // its chunks' maxima fit the LDS
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;
constexpr float kFarBelow = -1000.f;  // exp and 2 to the power of it are 0

struct LogprobArgs {
  const void *logits;
  int64_t row_stride;  // elements
  const void *tokens;  // nullable; int32 or int64
  int tokens64;
  int vocab, top;
  int slices, slice_len;  // elements, a multiple of kThreads * 8
  float *logprobs;
  int32_t *ranks;
  float *entropy;  // nullable
  int64_t *top_ids;
  int64_t ids_stride;
  float *top_logprobs;
  int64_t lps_stride;
  char *ws;  // slices > 1: [row][slice] a Part and `top` Listed
};

// What a slice says of its row: the largest logit, the sums of the others against
// it (see Sums), and how many of its tokens are ahead of the given one.
struct Part {
  float m, rest, mean;
  int before;
};
struct Listed {
  float x;
  int i;
};

__host__ __device__ inline int64_t part_bytes(int top) {
  return static_cast<int64_t>(sizeof(Part)) + top * static_cast<int64_t>(sizeof(Listed));
}

// A logit that is NaN counts as minus infinity.
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x; }

// Whether (x, i) comes ahead of (y, j).
__device__ __forceinline__ bool ahead(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

// A NaN of either kind gives way to the other operand of a maximum.  (In the mode that
// kernels begin in, a signalling one makes the result NaN, and as an instruction of three
// is two maxima, the second then drops what the first should have kept.)  The wave's
// MODE bit for it, cleared ahead of all loads, so ahead of the maxima over them.
__device__ __forceinline__ void nan_gives_way() {
  asm volatile("s_setreg_imm32_b32 hwreg(HW_REG_MODE, 9, 1), 0" ::: "memory");
}
// The largest of three, without the compiler's quieting of each operand: NaN only if all
// are, once nan_gives_way() was called.
__device__ __forceinline__ float max3_raw(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// The next larger value of fp32 (x not NaN or plus infinity).
__device__ __forceinline__ float next_above(float x) {
  const int b = __float_as_int(x + 0.f);
  return x == 0.f ? __int_as_float(1) : __int_as_float(b + (b < 0 ? -1 : 1));
}

// Sums over a set of logits with largest element m: r = sum exp(y) and q = sum y
// exp(y), y = x - m, over all but one element of value m.
struct Sums {
  float m, r, q;  // m = -inf: the set is empty
};
// The sums against a larger maximum.  `own`: this holder counts the element left out.
__device__ __forceinline__ void raise(Sums &s, float m, bool own) {
  if (s.m == m) return;
  if (s.m > -INFINITY) {
    const float d = m == INFINITY ? kFarBelow : fmaxf(s.m - m, kFarBelow);
    const float f = __builtin_amdgcn_exp2f(d * kLog2e);
    s.r += own ? 1.f : 0.f;
    s.q = f > 0.f ? (s.q + d * s.r) * f : 0.f;
    s.r *= f;
  }
  s.m = m;
}
// Two disjoint sets as one.
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  if (a.m < b.m) {
    const Sums t = a;
    a = b;
    b = t;
  }
  const bool tie = a.m == b.m && a.m > -INFINITY;
  raise(b, a.m, true);
  a.r += b.r + (tie ? 1.f : 0.f);
  a.q += b.q;
  return a;
}

// The sums as a wave forms them, its maximum m in every lane: in powers of two
// against m2, the fp32 value of m log2(e), so that an element takes one fma, t = x
// log2(e) - m2.  m itself then has t = off, some 2^-24 of m2, which `sums_of` takes out
// by 2^off = 1 + off ln 2: below 4096 |off| is 2^-12 at most and the square left out
// (off ln 2)^2 / 2 < 2^-26.  From there on (`far`, infinities too) t is (x - m) log2(e),
// a subtraction more an element, with m2 and off 0.
struct WaveSums {
  float m, m2, off;
  float r, q;  // sum 2^t, sum t 2^t, of the lane
};
__device__ __forceinline__ bool far(float m) { return !(fabsf(m) < 4096.f); }
// `own`: this lane counts the element left out so far.
__device__ __forceinline__ void raise(WaveSums &s, float m, bool own) {
  const float m2 = far(m) ? 0.f : m * kLog2e;
  const float off = far(m) ? 0.f : fmaf(m, kLog2e, -m2);
  if (s.m > -INFINITY) {
    const float d = fmaxf(fmaf(s.m - m, kLog2e, off - s.off), kFarBelow);
    const float f = __builtin_amdgcn_exp2f(d);
    const float w = own ? fmaf(s.off, kLn2, 1.f) : 0.f;  // 2^off
    s.r += w;
    s.q = fmaf(d, s.r, fmaf(s.off, w, s.q)) * f;
    s.r *= f;
  }
  s.m = m;
  s.m2 = m2;
  s.off = off;
}
__device__ __forceinline__ Sums sums_of(const WaveSums &s, float r, float q) {
  const float f = fmaf(-s.off, kLn2, 1.f);  // 2^-off
  return {s.m, r * f, fmaf(-s.off, r, q) * f * kLn2};
}

__device__ __forceinline__ float wave_sum_f32(float x) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) x += __shfl_xor(x, m, kWave);
  return x;
}

// Max over eight consecutive lanes, without the LDS (x not NaN).  A lane's value is
// read two states after it was written at the earliest, which the compiler, not
// looking into the statement, does not see to.
__device__ __forceinline__ float max_of_8(float x) {
  asm("s_nop 4\n\tv_max_f32_dpp %0, %0, %0 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf"
      : "+v"(x));
  return x;
}

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  T x[N];
};
// Elements at .. at + N - 1 of a row; those from `end` on read as minus infinity.
template <typename T>
__device__ __forceinline__ void load_vec(const T *row, int at, int end, Vec<T> &v) {
  if (at + Vec<T>::N <= end) {
    __builtin_memcpy(v.x, row + at, 16);
  } else {
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i) v.x[i] = at + i < end ? row[at + i] : static_cast<T>(-INFINITY);
  }
}

struct Shared {
  Part part[kWaves];
  float best[kThreads];
  Listed list[kMaxListed];
  Listed picked[kMaxTop], final[kMaxTop];
  float red_x[kWaves];
  int red_i[kWaves];
  int count;
  float floor;
};

// The foremost of the work-group's pairs, the same for every thread.
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
    sh.red_x[threadIdx.x / kWave] = x;
    sh.red_i[threadIdx.x / kWave] = i;
  }
  __syncthreads();
  x = sh.red_x[0];
  i = sh.red_i[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w)
    if (ahead(sh.red_x[w], sh.red_i[w], x, i)) {
      x = sh.red_x[w];
      i = sh.red_i[w];
    }
}

// A value that at least `want` of the work-group's threads' maxima reach: the largest
// of 16 bits (minus infinity if there is none).  Clears sh.count.
__device__ float floor_of(float best, int want, Shared &sh) {
  const int t = threadIdx.x;
  sh.best[t] = best;
  if (t == 0) sh.count = 0;
  __syncthreads();
  if (t < kWave) {
    // Bit by bit, as ordered integers, so that a bit set is a larger value.
    uint32_t key[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int bits = __float_as_int(sh.best[w * kWave + t] + 0.f);
      key[w] = static_cast<uint32_t>(bits < 0 ? ~bits : bits | static_cast<int>(0x80000000u));
    }
    uint32_t floor = 0;
#pragma unroll
    for (int b = 31; b >= 16; --b) {
      const uint32_t f = floor | 1u << b;
      int reach = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) reach += __popcll(__ballot(key[w] >= f));
      if (reach >= want) floor = f;
    }
    const int back = floor & 0x80000000u ? static_cast<int>(floor & 0x7FFFFFFFu) : ~static_cast<int>(floor);
    const float value = __int_as_float(back);
    if (t == 0) sh.floor = value == value ? value : -INFINITY;  // (below minus infinity the bits are a NaN's)
  }
  __syncthreads();
  return sh.floor;
}

// The foremost `want` of the pairs that each(take) names to every thread in turn, as
// take(value, id), into `out`, in order, and their number (fewer where the others are
// minus infinity); `best` is the largest value named to the thread.  Every thread
// calls it.  The floor leaves few pairs to rank; where too many reach it (ties), they
// are taken one at a time.
template <typename Each>
__device__ int foremost(float best, int want, Each each, Listed *out, Shared &sh) {
  const int t = threadIdx.x;
  const float floor = floor_of(best, want, sh);
  each([&](float v, int id) {
    if (v >= floor && v > -INFINITY) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kMaxListed) sh.list[at] = {v, id};
    }
  });
  __syncthreads();
  const int listed = sh.count;
  if (listed <= kMaxListed) {
    if (t < listed) {
      const Listed mine = sh.list[t];
      int rank = 0;
      for (int j = 0; j < listed; ++j) rank += ahead(sh.list[j].x, sh.list[j].i, mine.x, mine.i);
      if (rank < want) out[rank] = mine;
    }
    __syncthreads();
    return min(listed, want);
  }
  float last = INFINITY;
  int ilast = -1;
  for (int k = 0; k < want; ++k) {
    float v = -INFINITY;
    int i = INT32_MAX;
    each([&](float y, int j) {
      if (ahead(last, ilast, y, j) && ahead(y, j, v, i)) {
        v = y;
        i = j;
      }
    });
    block_first(v, i, sh);
    if (!(v > -INFINITY)) {
      __syncthreads();
      return k;
    }
    if (t == 0) out[k] = {v, i};
    last = v;
    ilast = i;
  }
  __syncthreads();
  return want;
}
// The same of n pairs (x(e), id(e)).
template <typename X, typename I>
__device__ int foremost_of(int n, int want, X x, I id, Listed *out, Shared &sh) {
  float best = -INFINITY;
  for (int e = threadIdx.x; e < n; e += kThreads) best = fmaxf(best, x(e));
  return foremost(
      best, want,
      [&](auto take) {
        for (int e = threadIdx.x; e < n; e += kThreads) take(x(e), id(e));
      },
      out, sh);
}

struct Result {
  float m, log_s, entropy;
  bool some;
};
__device__ __forceinline__ Result result_of(const Sums &s) {
  Result r;
  r.m = s.m;
  r.some = s.m > -INFINITY;
  const double log_s = log1p(static_cast<double>(s.r));
  r.log_s = static_cast<float>(log_s);
  r.entropy = r.some ? static_cast<float>(log_s - static_cast<double>(s.q) / (1.0 + s.r)) : 0.f;
  return r;
}
__device__ __forceinline__ float logprob_of(const Result &r, float x) {
  return r.some && x > -INFINITY ? (x == r.m ? 0.f : x - r.m) - r.log_s : -INFINITY;
}

__device__ __forceinline__ int64_t token_of(const LogprobArgs &a, int64_t row) {
  if (!a.tokens) return -1;
  return a.tokens64 ? static_cast<const int64_t *>(a.tokens)[row] : static_cast<const int32_t *>(a.tokens)[row];
}
template <typename T>
__device__ __forceinline__ float token_logit(const LogprobArgs &a, int64_t row, int64_t token) {
  if (token < 0 || token >= a.vocab) return -INFINITY;
  return clean(static_cast<float>(static_cast<const T *>(a.logits)[row * a.row_stride + token]));
}
template <typename T>
__device__ __forceinline__ void write_row(const LogprobArgs &a, int64_t row, const Result &r, int before, float xt) {
  if (a.tokens) {
    a.logprobs[row] = logprob_of(r, xt);
    a.ranks[row] = xt > -INFINITY ? before + 1 : 0;
  }
  if (a.entropy) a.entropy[row] = r.entropy;
}

__device__ __forceinline__ void write_top(const LogprobArgs &a, int64_t row, const Result &r, int found, const Shared &sh) {
  const int t = threadIdx.x;
  if (t >= a.top) return;
  a.top_ids[row * a.ids_stride + t] = t < found ? sh.final[t].i : -1;
  a.top_logprobs[row * a.lps_stride + t] = t < found ? logprob_of(r, sh.final[t].x) : -INFINITY;
}

// A slice of a row.  Every thread takes kStream 16-byte vectors of as many runs at a
// time, the next ones under way; HELD: the slice is one batch of HELD elements a
// thread, which stay in registers until the likeliest tokens are found.  (Such a call
// runs its code once, and most of its time is the code's way from memory: as few
// elements a thread as the slice needs.)
template <typename T, int HELD>
__global__ __launch_bounds__(kThreads) void logprob_kernel(LogprobArgs a) {
  constexpr int N = Vec<T>::N, kBatch = HELD ? HELD / N : kStream;
  constexpr bool ONE = HELD != 0;
  constexpr int CHUNK = kGroupLanes * N;  // elements, 128 bytes
  constexpr int STEP = kThreads * N;      // elements of one vector of every thread
  __shared__ Shared sh;
  extern __shared__ float values[];  // the largest of each chunk, later the picked chunks' tokens (ONE: not used)
  nan_gives_way();
  const int t = threadIdx.x, lane = t & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const int64_t row = blockIdx.x / static_cast<unsigned>(a.slices);
  const int slice = static_cast<int>(blockIdx.x - row * a.slices);
  const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
  const int first = slice * a.slice_len;
  const int end = static_cast<int>(min(static_cast<int64_t>(first) + a.slice_len, static_cast<int64_t>(a.vocab)));

  Vec<T> v[kBatch];
  auto load = [&](int at) __attribute__((always_inline)) {
    if (at + kBatch * STEP <= end) {  // the same for all threads
#pragma unroll
      for (int j = 0; j < kBatch; ++j) __builtin_memcpy(v[j].x, x + at + j * STEP + t * N, 16);
    } else {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) load_vec(x, at + j * STEP + t * N, end, v[j]);
    }
  };
  load(first);
  const int64_t token = token_of(a, row);
  const float xt = token_logit<T>(a, row, token);
  // Ahead of the token: at lower indices what is not less, at higher ones what is larger.
  const float above = xt < INFINITY ? next_above(xt) : NAN;  // nothing is larger than plus infinity
  const bool ranked = xt > -INFINITY;

  WaveSums s = {-INFINITY, 0.f, 0.f, 0.f, 0.f};
  int before = 0;  // tokens ahead: of the wave, in scalars
  int mixed = 0;   // of the lane, in the run that holds the token
  float f[kBatch][N], vmax[kBatch];
  for (int at = first; at < end; at += kBatch * STEP) {
    bool usual = true;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[j][i] = static_cast<float>(v[j].x[i]);
      float mx = max3_raw(f[j][0], f[j][1], f[j][2]);
#pragma unroll
      for (int i = 3; i + 1 < N; i += 2) mx = max3_raw(mx, f[j][i], f[j][i + 1]);
      vmax[j] = max3_raw(mx, f[j][N - 1], f[j][N - 1]);
      usual &= vmax[j] <= s.m;  // false for NaN
    }
    if (!ONE && at + kBatch * STEP < end) load(at + kBatch * STEP);
    const bool special = !__all(usual) || far(s.m);
    bool holder = false;  // of a new maximum, whose first element is left out of the sums
    if (special) {
      // A new maximum, a vector of NaN, or nothing so far.
      bool nan = ONE;  // (the elements are needed without NaN)
#pragma unroll
      for (int j = 0; j < kBatch; ++j) nan |= vmax[j] != vmax[j];
      if (__any(nan)) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          vmax[j] = -INFINITY;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            f[j][i] = clean(f[j][i]);
            vmax[j] = fmaxf(vmax[j], f[j][i]);
          }
        }
      }
      float mine = vmax[0];
#pragma unroll
      for (int j = 1; j < kBatch; ++j) mine = fmaxf(mine, vmax[j]);
      float m = mine;
#pragma unroll
      for (int d = 1; d < kWave; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, kWave));
      if (m > s.m) {
        raise(s, m, lane == 0);
        holder = lane == __builtin_ctzll(__ballot(mine == m));
      }
    }
    if (ranked) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int w0 = at + j * STEP + wave * kWave * N;  // the wave's first element
        if (w0 + kWave * N <= token || w0 > token) {
          const float bar = w0 > token ? above : xt;
#pragma unroll
          for (int i = 0; i < N; ++i) before += __popcll(__ballot(f[j][i] >= bar));
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) mixed += f[j][i] >= (w0 + lane * N + i < token ? xt : above);
        }
      }
    }
    if (!ONE && a.top) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const float c = max_of_8(vmax[j]);
        if ((lane & (kGroupLanes - 1)) == 0) values[(at - first + j * STEP + t * N) / CHUNK] = c;
      }
    }
    auto add = [&](float t, float &r, float &q) __attribute__((always_inline)) {
      const float y = fmaxf(t, kFarBelow);  // a NaN or minus infinity: 2^y is 0
      const float e = __builtin_amdgcn_exp2f(y);
      r += e;
      q = fmaf(y, e, q);
    };
    if (!special) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        float r = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) add(fmaf(f[j][i], kLog2e, -s.m2), r, q);
        s.r += r;
        s.q += q;
      }
    } else if (s.m > -INFINITY) {
      const float base = far(s.m) ? s.m : 0.f;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        float r = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const bool equal = f[j][i] == s.m;
          if (holder && equal)
            holder = false;
          else
            add(equal ? s.off : fmaf(f[j][i] - base, kLog2e, -s.m2), r, q);  // (equal: of infinities no difference)
        }
        s.r += r;
        s.q += q;
      }
    }
  }
  const float r = wave_sum_f32(s.r), q = wave_sum_f32(s.q);
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) mixed += __shfl_xor(mixed, m, kWave);
  if (lane == 0) {
    const Sums w = sums_of(s, r, q);
    sh.part[wave] = {w.m, w.r, w.q, before + mixed};
  }
  __syncthreads();
  Sums sum = {sh.part[0].m, sh.part[0].rest, sh.part[0].mean};
  before = sh.part[0].before;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    sum = join(sum, {sh.part[w].m, sh.part[w].rest, sh.part[w].mean});
    before += sh.part[w].before;
  }

  int found = 0;
  if (a.top) {
    if constexpr (ONE) {
      float best = -INFINITY;
      if (first < end) {
        best = vmax[0];
#pragma unroll
        for (int j = 1; j < kBatch; ++j) best = fmaxf(best, vmax[j]);
      }
      found = foremost(
          best, a.top,
          [&](auto take) {
            if (first >= end) return;
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
#pragma unroll
              for (int i = 0; i < N; ++i) take(f[j][i], first + j * STEP + t * N + i);
          },
          sh.final, sh);
    } else {
      // The foremost `top` chunks hold the foremost `top` tokens: a token of another
      // chunk has the largest of each of them ahead of it, chunks being runs of tokens.
      const int chunks = (max(end - first, 0) + CHUNK - 1) / CHUNK;
      const int picked = foremost_of(chunks, a.top, [&](int e) { return values[e]; }, [](int e) { return e; }, sh.picked, sh);
      for (int e = t; e < picked * kGroupLanes; e += kThreads) {
        Vec<T> w;
        load_vec(x, first + sh.picked[e / kGroupLanes].i * CHUNK + e % kGroupLanes * N, end, w);
#pragma unroll
        for (int i = 0; i < N; ++i) values[e * N + i] = clean(static_cast<float>(w.x[i]));
      }
      __syncthreads();
      found = foremost_of(
          picked * CHUNK, a.top, [&](int e) { return values[e]; },
          [&](int e) { return first + sh.picked[e / CHUNK].i * CHUNK + e % CHUNK; }, sh.final, sh);
    }
  }
  if (a.slices == 1) {
    const Result res = result_of(sum);
    if (t == 0) write_row<T>(a, row, res, before, xt);
    write_top(a, row, res, found, sh);
    return;
  }
  char *out = a.ws + blockIdx.x * part_bytes(a.top);
  if (t == 0) *reinterpret_cast<Part *>(out) = {sum.m, sum.r, sum.q, before};
  if (t < a.top) reinterpret_cast<Listed *>(out + sizeof(Part))[t] = t < found ? sh.final[t] : Listed{-INFINITY, INT32_MAX};
}

// Joins the slices of one row.
template <typename T>
__global__ __launch_bounds__(kThreads) void logprob_join_kernel(LogprobArgs a) {
  __shared__ Shared sh;
  extern __shared__ float values[];  // slices * top values, then their tokens
  const int t = threadIdx.x, lane = t & (kWave - 1);
  const int64_t row = blockIdx.x;
  const float xt = token_logit<T>(a, row, token_of(a, row));
  const char *parts = a.ws + row * a.slices * part_bytes(a.top);
  const int n = a.slices * a.top;
  int *ids = reinterpret_cast<int *>(values + n);
  for (int e = t; e < n; e += kThreads) {
    const int slice = e / a.top;
    const Listed l = reinterpret_cast<const Listed *>(parts + slice * part_bytes(a.top) + sizeof(Part))[e - slice * a.top];
    values[e] = l.x;
    ids[e] = l.i;
  }
  Part p = {-INFINITY, 0.f, 0.f, 0};
  if (lane < a.slices) p = *reinterpret_cast<const Part *>(parts + lane * part_bytes(a.top));
  Sums s = {p.m, p.rest, p.mean};
  int before = p.before;
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    const Sums o = {__shfl_xor(s.m, m, kWave), __shfl_xor(s.r, m, kWave), __shfl_xor(s.q, m, kWave)};
    s = join(s, o);
    before += __shfl_xor(before, m, kWave);
  }
  __syncthreads();
  const int found = a.top ? foremost_of(n, a.top, [&](int e) { return values[e]; }, [&](int e) { return ids[e]; }, sh.final, sh) : 0;
  const Result r = result_of(s);
  if (t == 0) write_row<T>(a, row, r, before, xt);
  write_top(a, row, r, found, sh);
}

// How many slices a row is cut into.  One that a work-group holds, or nearly, is not
// cut (256 x 8000 bf16 11.4 us in one launch, 16.8 in slices and a second one).  Others
// are for two work-groups a compute unit, or for four where that leaves slices that
// are held in few registers, or long ones.  Measured, two a unit / four, us: 48 x 65537
// fp16 17.0 / 15.7, 128 x 32000 fp32 22.4 / 18.8, 256 x 32000 bf16 25.5 / 28.5, 512 x
// 32000 bf16 26.0 / 30.8, 128 x 152000 fp32 38.1 / 35.0, 256 x 152000 bf16 48.7 / 44.1
// (one: 53.0; eight: 56.7).
constexpr int64_t kHeldWhole = 8192, kShortSlice = 4096, kLongSlice = 16384;
int slices_of(int64_t rows, int64_t vocab) {
  if (vocab <= kHeldWhole) return 1;
  const int64_t units = device_cus();
  const int64_t four = (4 * units + rows - 1) / rows, two = (2 * units + rows - 1) / rows;
  const int64_t wanted = vocab <= four * kShortSlice || vocab >= four * kLongSlice ? four : two;
  const int64_t most = (vocab + kSliceUnit - 1) / kSliceUnit;
  const int64_t least = (vocab + kMaxSliceLen - 1) / kMaxSliceLen;
  int64_t n = wanted < most ? wanted : most;
  n = n < kMaxSlices ? n : kMaxSlices;
  return static_cast<int>(n > least ? n : least);
}

template <typename T>
int launch(LogprobArgs a, int64_t rows, hipStream_t s) {
  constexpr int CHUNK = kGroupLanes * Vec<T>::N, ROUND = kStream * kThreads * Vec<T>::N;
  const dim3 grid(static_cast<unsigned>(rows * a.slices)), block(kThreads);
  if (a.slice_len <= 8 * kThreads) {
    logprob_kernel<T, 8><<<grid, block, 0, s>>>(a);
  } else if (a.slice_len <= 16 * kThreads) {
    logprob_kernel<T, 16><<<grid, block, 0, s>>>(a);
  } else if (a.slice_len <= 32 * kThreads && sizeof(T) == 2) {
    logprob_kernel<T, sizeof(T) == 2 ? 32 : 16><<<grid, block, 0, s>>>(a);
  } else {
    const int64_t chunks = static_cast<int64_t>((a.slice_len + ROUND - 1) / ROUND) * ROUND / CHUNK;
    const int64_t floats = !a.top ? 0 : chunks > a.top * CHUNK ? chunks : a.top * CHUNK;
    logprob_kernel<T, 0><<<grid, block, floats * 4, s>>>(a);
  }
  int rc = launch_status("k8v4_token_logprobs");
  if (rc || a.slices == 1) return rc;
  logprob_join_kernel<T><<<dim3(static_cast<unsigned>(rows)), dim3(kThreads), a.slices * a.top * 8, s>>>(a);
  return launch_status("k8v4_token_logprobs join");
}

constexpr int64_t kMaxVocab = int64_t(1) << 24;
constexpr int64_t kMaxGroups = int64_t(1) << 24;  // work-groups of a launch, 2^32 threads

}  // namespace
}  // namespace k8v4

extern "C" int64_t k8v4_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int top) {
  using namespace k8v4;
  if (rows < 0 || vocab < 1 || vocab > kMaxVocab || top < 0 || top > kMaxTop) return -1;
  const int64_t slices = rows ? slices_of(rows, vocab) : 1;
  if (rows >= kMaxGroups / slices) return -1;
  return slices == 1 ? 0 : rows * slices * part_bytes(top);
}

extern "C" int k8v4_token_logprobs(const void *logits, int dtype, int64_t row_stride, const void *tokens,
                                   int tokens_are_int64, int64_t rows, int64_t vocab, int top, float *logprobs,
                                   int32_t *ranks, float *entropy, int64_t *top_ids, int64_t ids_stride,
                                   float *top_logprobs, int64_t lps_stride, void *workspace, int64_t workspace_bytes,
                                   void *stream) {
  using namespace k8v4;
  clear_error();
  K8V4_REQUIRE(dtype == K8V4_F16 || dtype == K8V4_BF16 || dtype == K8V4_F32, "logits must be fp16, bf16 or fp32");
  K8V4_REQUIRE(rows >= 0, "negative number of rows");
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
  K8V4_REQUIRE(need >= 0, "too many rows for one launch");
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
  a.vocab = static_cast<int>(vocab);
  a.top = top;
  a.logprobs = logprobs;
  a.ranks = ranks;
  a.entropy = entropy;
  a.top_ids = top_ids;
  a.ids_stride = ids_stride;
  a.top_logprobs = top_logprobs;
  a.lps_stride = lps_stride;
  a.slices = slices_of(rows, vocab);
  a.slice_len = static_cast<int>(((vocab + a.slices - 1) / a.slices + kSliceUnit - 1) / kSliceUnit * kSliceUnit);
  a.ws = static_cast<char *>(workspace);
  auto s = static_cast<hipStream_t>(stream);
  if (dtype == K8V4_F32) return launch<float>(a, rows, s);
  return dtype == K8V4_BF16 ? launch<__bf16>(a, rows, s) : launch<_Float16>(a, rows, s);
}
