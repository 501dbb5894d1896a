// Cache rows of the accepted branch of a drafted tree moved to the places of a
// linear sequence.  No counterpart in the reference, whose drafts are chains.
//
// Sequence b's tree was stored from token s_b on, node n at token s_b + n; node
// path[b][i] is the i-th of the branch.  Token s_b + path[b][i] is copied to token
// s_b + i, codes and planes as they are, for i = 0 .. accepted[b].
//
// path[i] >= i (a branch's i-th node has i ancestors ahead of it; other entries
// move nothing), so what step i reads is never what an earlier step wrote, and
// taking the steps in order gives what reading everything first would.  A thread
// owns a slice of a token's row in one region (16 bytes of K, 8 of V, a word of a
// plane) and moves that slice of every node itself, eight nodes' loads in flight,
// so no two threads touch the same bytes and nothing has to be waited for.  The
// slots are found once for all of them, by one wave, a lane an entry.
//
// Bound by latency: a branch is a few rows of 1 to 2 KB, found by three dependent
// loads (path, table, row): one branch of a 13-node tree takes 4.0 us, 128 of 26-node
// trees (head dim 256) 6.4.
#include "k8v4_common.h"

namespace k8v4 {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct KeepArgs {
  char *base[5];   // k, k_scale, v, v_scale, v_zero
  int64_t ps[5];   // page strides, bytes
  int64_t num_pages;
  const int32_t *block_table;
  int64_t bt_stride;
  int64_t table_pages;
  int ppb;
  const int32_t *starts, *path, *accepted;
  int64_t path_stride;
  int width;  // entries of a path row
  int hkv, head_dim;
};

constexpr int kThreads = 192;  // slices of a token at most: 64 of K, 64 of V, 12 of the planes
constexpr int kInFlight = 8;
constexpr int kEntries = kWave;  // looked up together

// Slot (page * 64 + row) of token t, -1 if it has none.
__device__ __forceinline__ int64_t slot_of(const KeepArgs &a, const int32_t *row, int64_t t) {
  if (t < 0 || t >= a.table_pages * kPage) return -1;
  const uint32_t p = static_cast<uint32_t>(t / kPage), ppb = static_cast<uint32_t>(a.ppb);
  const uint32_t entry = ppb == 1 ? p : p / ppb;
  const int64_t page = static_cast<int64_t>(row[entry]) * a.ppb + (p - entry * ppb);
  return page >= 0 && page < a.num_pages ? page * kPage + t % kPage : -1;
}

struct Move {
  int64_t from, to;  // slots
};

template <typename T>
__device__ __forceinline__ void move_slice(char *base, int64_t ps, int row_bytes, int off, const Move *moves, int count) {
  for (int i0 = 0; i0 < count; i0 += kInFlight) {
    T x[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int64_t s = moves[min(i0 + u, count - 1)].from;
      x[u] = *reinterpret_cast<const T *>(base + (s >> 6) * ps + (s & 63) * row_bytes + off);
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (i0 + u >= count) break;
      const int64_t s = moves[i0 + u].to;
      *reinterpret_cast<T *>(base + (s >> 6) * ps + (s & 63) * row_bytes + off) = x[u];
    }
  }
}

__global__ __launch_bounds__(kThreads) void kv_keep_kernel(KeepArgs a) {
  __shared__ Move moves[kEntries];
  __shared__ int count;
  const int b = blockIdx.x, t = threadIdx.x;
  const int k_row = a.hkv * a.head_dim, v_row = k_row / 2, plane_row = a.hkv * 4;
  const int nk = k_row / 16, nv = v_row / 8;
  const int kept = min(max(a.accepted[b], -1), a.width - 1) + 1;
  for (int i0 = 0; i0 < kept; i0 += kEntries) {
    if (t < kEntries) {
      const int i = i0 + t;
      const int node = i < kept ? a.path[b * a.path_stride + i] : -1;
      const int32_t *row = a.block_table + b * a.bt_stride;
      const int64_t first = a.starts[b];
      Move m = {-1, -1};
      if (node > i) m = {slot_of(a, row, first + node), slot_of(a, row, first + i)};
      const bool moves_it = m.from >= 0 && m.to >= 0;
      const uint64_t all = __ballot(moves_it);
      if (moves_it) moves[__popcll(all & ((uint64_t(1) << t) - 1))] = m;
      if (t == 0) count = __popcll(all);
    }
    __syncthreads();
    const int n = count;
    if (t < nk) {
      move_slice<u32x4>(a.base[0], a.ps[0], k_row, 16 * t, moves, n);
    } else if (t < nk + nv) {
      move_slice<uint64_t>(a.base[2], a.ps[2], v_row, 8 * (t - nk), moves, n);
    } else if (t < nk + nv + 3 * a.hkv) {
      const int p = (t - nk - nv) / a.hkv, r = p == 0 ? 1 : p + 2;
      move_slice<uint32_t>(a.base[r], a.ps[r], plane_row, 4 * ((t - nk - nv) % a.hkv), moves, n);
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace k8v4

extern "C" int k8v4_kv_keep_paged(int8_t *k_cache, float *k_scale, uint8_t *v_cache, float *v_scale, float *v_zero,
                                  int64_t num_pages, int64_t k_page_stride, int64_t ks_page_stride,
                                  int64_t v_page_stride, int64_t vs_page_stride, int64_t vz_page_stride,
                                  const int32_t *block_table, int64_t bt_stride, int64_t table_width,
                                  int pages_per_block, const int32_t *seq_starts, const int32_t *path,
                                  int64_t path_stride, int width, const int32_t *accepted, int64_t batch, int hkv,
                                  int head_dim, void *stream) {
  using namespace k8v4;
  clear_error();
  K8V4_REQUIRE(supported_heads(hkv), "unsupported per-GPU KV head count %d (this library serves 2 or 4)", hkv);
  K8V4_REQUIRE(supported_dim(head_dim), "unsupported head dim %d (this library serves 128 or 256)", head_dim);
  K8V4_REQUIRE(pages_per_block >= 1, "pages_per_block");
  K8V4_REQUIRE(num_pages >= 1 && num_pages <= INT32_MAX, "num_pages must be 1 .. 2^31 - 1");
  K8V4_REQUIRE(batch >= 0 && batch < (int64_t(1) << 24), "bad batch");
  K8V4_REQUIRE(width >= 0, "negative path width");
  if (batch == 0 || width == 0) return K8V4_OK;
  K8V4_REQUIRE(table_width >= 1 && table_width <= (int64_t(1) << 30) / pages_per_block, "block_table width");
  K8V4_REQUIRE(k_cache && k_scale && v_cache && v_scale && v_zero && block_table && seq_starts && path && accepted,
               "null pointer");
  const auto aligned = [](const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  K8V4_REQUIRE(bt_stride >= table_width || batch == 1, "block_table row stride shorter than its width");
  K8V4_REQUIRE(path_stride >= width || batch == 1, "path row stride shorter than its width");
  K8V4_REQUIRE(aligned(block_table, 4) && aligned(seq_starts, 4) && aligned(path, 4) && aligned(accepted, 4),
               "index arrays misaligned");
  K8V4_REQUIRE(aligned(k_cache, 16) && aligned(k_scale, 4) && aligned(v_cache, 8) && aligned(v_scale, 4) &&
                   aligned(v_zero, 4),
               "cache region misaligned");
  K8V4_REQUIRE(k_page_stride % 16 == 0 && ks_page_stride % 4 == 0 && v_page_stride % 8 == 0 &&
                   vs_page_stride % 4 == 0 && vz_page_stride % 4 == 0,
               "cache page strides must keep rows aligned");
  KeepArgs a = {};
  a.base[0] = reinterpret_cast<char *>(k_cache);
  a.base[1] = reinterpret_cast<char *>(k_scale);
  a.base[2] = reinterpret_cast<char *>(v_cache);
  a.base[3] = reinterpret_cast<char *>(v_scale);
  a.base[4] = reinterpret_cast<char *>(v_zero);
  a.ps[0] = k_page_stride;
  a.ps[1] = ks_page_stride;
  a.ps[2] = v_page_stride;
  a.ps[3] = vs_page_stride;
  a.ps[4] = vz_page_stride;
  a.num_pages = num_pages;
  a.block_table = block_table;
  a.bt_stride = bt_stride;
  a.table_pages = table_width * pages_per_block;
  a.ppb = pages_per_block;
  a.starts = seq_starts;
  a.path = path;
  a.accepted = accepted;
  a.path_stride = path_stride;
  a.width = width;
  a.hkv = hkv;
  a.head_dim = head_dim;
  kv_keep_kernel<<<dim3(static_cast<unsigned>(batch)), dim3(kThreads), 0, static_cast<hipStream_t>(stream)>>>(a);
  return launch_status("k8v4_kv_keep_paged");
}
