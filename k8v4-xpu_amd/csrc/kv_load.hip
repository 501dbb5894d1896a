// Reading the paged cache back: int8 K codes and packed int4 V codes of a
// ragged batch of token ranges -> contiguous fp16, bf16 or fp32 rows.
//
// Row r of the outputs belongs to the sequence b with row_starts[b] <= r <
// row_starts[b + 1] and holds its token t = seq_starts[b] + r - row_starts[b]:
//   K[d] = code[d] * k_scale,   V[d] = (nibble[d] - v_zero) * v_scale
// (the dequantization rule of k8v4_v030/dequant.py:96-106), each a product in
// fp32 rounded to nearest once more into a 16-bit output.
//
// Bound by memory: hkv * (1.5 D + 12) bytes read and 4 hkv D (16-bit) or
// 8 hkv D (fp32) written per token, a handful of vector instructions per
// eight dims.  A work-group takes kRows consecutive rows: its first kRows lanes
// look up each row's sequence and cache cell once, into LDS; then every thread
// converts eight dims of one (row, head) at a time, so the 64 lanes of a wave
// read contiguous codes and write a contiguous kilobyte (fp32: two kilobytes by
// two stores of every other 16 bytes each).
//
// A small call is a chain of round trips: starts, first token, table entry, then
// the passes.  The search for a row's sequence runs over 256 of row_starts in LDS,
// read in one of them (a binary search of the array itself is one for each
// halving); only batches of more than 256 sequences search the array for the rest.
// Sixteen rows a work-group are two to eight passes, one after the other: their
// branches keep a pass's K loads, K stores, V loads and V stores in that order,
// each load waited for before the store behind it, so a wave makes two round trips
// a pass and only the other waves of the CU fill them (in large calls they do).
//
// Measured on cold pages in random order, 16-bit outputs, by 16 rows a
// work-group (by 8, by 32): 500 rows of 4 heads 5.3 us (5.3, 7.3), 19,800 rows of
// 2 heads at head dim 256 from twelve sequences 12.8 (13.0, 13.5), 262,144 rows of
// 4 heads 154.6, 4.86 TB/s of codes read and rows written (164.1, 154.6); a copy
// of 1 GiB moves 5.0 TB/s.  fp32 outputs: 131,072 rows of 4 heads 179.8 us, 3.58
// TB/s (half-line stores), 500 rows 6.6.
#include "k8v4_common.h"

namespace k8v4 {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kRows = 16;  // rows of one work-group

struct LoadArgs {
  const int8_t *k_cache;
  const float *k_scale;
  const uint8_t *v_cache;
  const float *v_scale;
  const float *v_zero;
  int64_t num_pages;
  int64_t k_ps, ks_ps, v_ps, vs_ps, vz_ps;  // page strides, bytes
  const int32_t *block_table;
  int64_t bt_stride;
  int64_t capacity;  // tokens a table row covers
  int ppb;
  const int32_t *seq_starts;  // nullable: 0
  const int32_t *row_starts;  // [batch + 1]
  int batch;
  int64_t rows;  // rows of the outputs
  void *k_out;
  void *v_out;
  int64_t k_stride, v_stride;  // elements between output rows
  int k_vec, v_vec;            // 16-byte aligned rows: vector stores
  int do_k, do_v;
};

// Eight values to consecutive elements of type T.
template <typename T>
__device__ __forceinline__ void put8(void *out, int64_t at, bool vec, const f8 &x) {
  T *dst = static_cast<T *>(out) + at;
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<f4 *>(dst)[0] = (f4){x[0], x[1], x[2], x[3]};
      reinterpret_cast<f4 *>(dst)[1] = (f4){x[4], x[5], x[6], x[7]};
    } else {
      typedef T t8 __attribute__((ext_vector_type(8)));
      *reinterpret_cast<t8 *>(dst) = __builtin_convertvector(x, t8);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = static_cast<T>(x[i]);
  }
}

template <typename T, int D, int HKV>
__global__ __launch_bounds__(kThreads) void kv_load_kernel(LoadArgs a) {
  constexpr int UPR = HKV * D / 8;          // eight-dim units of a row: 32, 64 or 128
  constexpr int RPP = kThreads / UPR;       // rows of one pass
  constexpr int PASSES = kRows / RPP;
  __shared__ int starts[kThreads];  // every step-th of row_starts
  __shared__ int cell[kRows];        // row within the page, -1: zeros, -2: no row of any sequence
  __shared__ int page[kRows];
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRows;
  const int t = threadIdx.x;
  const int step = (a.batch + kThreads - 1) / kThreads;
  const int known = (a.batch + step - 1) / step;  // at most kThreads
  const int end = a.row_starts[a.batch];
  if (t < known) starts[t] = a.row_starts[t * step];
  __syncthreads();
  if (t < kRows) {
    const int64_t r = r0 + t;
    int c = -2, p = 0;
    if (r < a.rows && r >= starts[0] && r < end) {
      int lo = 0, hi = known;  // starts[lo] <= r < starts[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= r)
          lo = mid;
        else
          hi = mid;
      }
      int first = starts[lo];
      lo *= step;
      hi = min(lo + step, a.batch);  // row_starts[lo] <= r < row_starts[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        const int x = a.row_starts[mid];
        if (x <= r) {
          lo = mid;
          first = x;
        } else {
          hi = mid;
        }
      }
      const int64_t tok = r - first + (a.seq_starts ? a.seq_starts[lo] : 0);
      c = -1;
      if (tok >= 0 && tok < a.capacity) {
        const uint32_t lp = static_cast<uint32_t>(tok / kPage);  // page of the sequence, below 2^30
        const uint32_t e = a.ppb <= 1 ? lp : lp / static_cast<uint32_t>(a.ppb);
        const int64_t ph = static_cast<int64_t>(a.block_table[lo * a.bt_stride + e]) * a.ppb + (lp - e * a.ppb);
        if (ph >= 0 && ph < a.num_pages) {
          p = static_cast<int>(ph);
          c = static_cast<int>(tok % kPage);
        }
      }
    }
    cell[t] = c;
    page[t] = p;
  }
  __syncthreads();
  const int u = t % UPR, sub = t / UPR;
  const int head = u / (D / 8), col = 8 * (u - head * (D / 8));
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int lr = i * RPP + sub;
    const int c = cell[lr];
    if (c == -2) continue;
    const int64_t p = page[lr];
    const int64_t r = r0 + lr;
    const bool live = c >= 0;
    const int64_t plane = static_cast<int64_t>(live ? c : 0) * HKV + head;
    if (a.do_k) {
      uint2 w = {0u, 0u};
      float s = 0.f;
      if (live) {
        w = *reinterpret_cast<const uint2 *>(reinterpret_cast<const char *>(a.k_cache) + p * a.k_ps + plane * D + col);
        s = *reinterpret_cast<const float *>(reinterpret_cast<const char *>(a.k_scale) + p * a.ks_ps + plane * 4);
      }
      f8 x;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = static_cast<float>(static_cast<int8_t>((e < 4 ? w.x : w.y) >> (8 * (e & 3)))) * s;
      put8<T>(a.k_out, r * a.k_stride + head * D + col, a.k_vec, x);
    }
    if (a.do_v) {
      uint32_t w = 0u;
      float s = 0.f, z = 0.f;
      if (live) {
        w = *reinterpret_cast<const uint32_t *>(reinterpret_cast<const char *>(a.v_cache) + p * a.v_ps +
                                                plane * (D / 2) + col / 2);
        s = *reinterpret_cast<const float *>(reinterpret_cast<const char *>(a.v_scale) + p * a.vs_ps + plane * 4);
        z = *reinterpret_cast<const float *>(reinterpret_cast<const char *>(a.v_zero) + p * a.vz_ps + plane * 4);
      }
      f8 x;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (static_cast<float>((w >> (4 * e)) & 15u) - z) * s;
      put8<T>(a.v_out, r * a.v_stride + head * D + col, a.v_vec, x);
    }
  }
}

template <typename T>
void launch(const LoadArgs &a, int hkv, int head_dim, hipStream_t s) {
  const dim3 blocks(static_cast<unsigned>((a.rows + kRows - 1) / kRows));
  if (head_dim == 128) {
    if (hkv == 4)
      kv_load_kernel<T, 128, 4><<<blocks, dim3(kThreads), 0, s>>>(a);
    else
      kv_load_kernel<T, 128, 2><<<blocks, dim3(kThreads), 0, s>>>(a);
  } else {
    if (hkv == 4)
      kv_load_kernel<T, 256, 4><<<blocks, dim3(kThreads), 0, s>>>(a);
    else
      kv_load_kernel<T, 256, 2><<<blocks, dim3(kThreads), 0, s>>>(a);
  }
}

bool aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace k8v4

extern "C" int k8v4_kv_load_paged(const int8_t *k_cache, const float *k_scale, const uint8_t *v_cache,
                                  const float *v_scale, const float *v_zero, int64_t num_pages,
                                  int64_t k_page_stride, int64_t ks_page_stride, int64_t v_page_stride,
                                  int64_t vs_page_stride, int64_t vz_page_stride, const int32_t *block_table,
                                  int64_t bt_stride, int64_t table_width, int pages_per_block,
                                  const int32_t *seq_starts, const int32_t *row_starts, int64_t batch, int hkv,
                                  int head_dim, void *k_out, void *v_out, int out_dtype, int64_t k_out_stride,
                                  int64_t v_out_stride, int64_t rows, void *stream) {
  using namespace k8v4;
  clear_error();
  const bool do_k = k_out != nullptr, do_v = v_out != nullptr;
  K8V4_REQUIRE(supported_heads(hkv), "unsupported per-GPU KV head count %d (this library serves 2 or 4)", hkv);
  K8V4_REQUIRE(supported_dim(head_dim), "unsupported head dim %d (this library serves 128 or 256)", head_dim);
  K8V4_REQUIRE(out_dtype == K8V4_F16 || out_dtype == K8V4_BF16 || out_dtype == K8V4_F32,
               "out dtype must be fp16, bf16 or fp32");
  K8V4_REQUIRE(pages_per_block >= 1, "pages_per_block");
  K8V4_REQUIRE(num_pages >= 1 && num_pages <= INT32_MAX, "num_pages must be 1 .. 2^31 - 1");
  K8V4_REQUIRE(batch >= 0 && batch < (1 << 24) && rows >= 0, "negative or too large batch or row count");
  K8V4_REQUIRE(do_k || do_v || rows == 0, "null pointer");
  if (batch == 0 || rows == 0) return K8V4_OK;
  K8V4_REQUIRE(table_width >= 1 && table_width <= (int64_t(1) << 30) / pages_per_block, "block_table width");
  K8V4_REQUIRE(bt_stride >= table_width || batch == 1, "block_table row stride shorter than its width");
  K8V4_REQUIRE(block_table && row_starts && (!do_k || (k_cache && k_scale)) &&
                   (!do_v || (v_cache && v_scale && v_zero)),
               "null pointer");
  const int64_t row = static_cast<int64_t>(hkv) * head_dim;
  K8V4_REQUIRE((!do_k || k_out_stride >= row) && (!do_v || v_out_stride >= row),
               "k/v row stride shorter than hkv*head_dim");
  K8V4_REQUIRE((!do_k || (aligned(k_cache, 16) && k_page_stride % 16 == 0)) &&
                   (!do_v || (aligned(v_cache, 8) && v_page_stride % 8 == 0)),
               "cache code rows must stay aligned");
  K8V4_REQUIRE((!do_k || (aligned(k_scale, 4) && ks_page_stride % 4 == 0)) &&
                   (!do_v || (aligned(v_scale, 4) && aligned(v_zero, 4) && vs_page_stride % 4 == 0 &&
                              vz_page_stride % 4 == 0)),
               "scale planes must be 4-byte aligned");
  K8V4_REQUIRE(aligned(block_table, 4) && aligned(row_starts, 4) && aligned(seq_starts, 4), "index arrays misaligned");
  const int esize = out_dtype == K8V4_F32 ? 4 : 2;
  K8V4_REQUIRE(aligned(k_out, esize) && aligned(v_out, esize), "k/v output misaligned");

  LoadArgs a;
  a.k_cache = k_cache;
  a.k_scale = k_scale;
  a.v_cache = v_cache;
  a.v_scale = v_scale;
  a.v_zero = v_zero;
  a.num_pages = num_pages;
  a.k_ps = k_page_stride;
  a.ks_ps = ks_page_stride;
  a.v_ps = v_page_stride;
  a.vs_ps = vs_page_stride;
  a.vz_ps = vz_page_stride;
  a.block_table = block_table;
  a.bt_stride = bt_stride;
  a.capacity = table_width * pages_per_block * kPage;
  a.ppb = pages_per_block;
  a.seq_starts = seq_starts;
  a.row_starts = row_starts;
  a.batch = static_cast<int>(batch);
  a.rows = rows;
  a.k_out = k_out;
  a.v_out = v_out;
  a.k_stride = k_out_stride;
  a.v_stride = v_out_stride;
  a.k_vec = aligned(k_out, 16) && k_out_stride * esize % 16 == 0;
  a.v_vec = aligned(v_out, 16) && v_out_stride * esize % 16 == 0;
  a.do_k = do_k;
  a.do_v = do_v;
  const int64_t blocks = (rows + kRows - 1) / kRows;
  K8V4_REQUIRE(blocks < (int64_t(1) << 31), "too many rows for one launch");
  auto s = static_cast<hipStream_t>(stream);
  if (out_dtype == K8V4_F32)
    launch<float>(a, hkv, head_dim, s);
  else if (out_dtype == K8V4_BF16)
    launch<__bf16>(a, hkv, head_dim, s);
  else
    launch<_Float16>(a, hkv, head_dim, s);
  return launch_status("k8v4_kv_load_paged");
}
