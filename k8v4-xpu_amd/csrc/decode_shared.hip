// Paged decode / MTP-verify attention of a batch whose sequences begin with
// the same cached pages, those read once for all of them.
//
// For every query row (token j of sequence b, query head) with visible end
// e = seq_len_b - q_len + j + 1, softmax attention over the keys t < e as in
// k8v4_attn_batch (int8-quantized query rows; exact integer dot products, whose
// scaling by k_scale is off by at most 0.75 of a unit of the dot; V as (nibble -
// zero) * scale), where the keys below P (the prefix's whole pages) are those of one
// table row and the others those of the sequence's own row.
// With the (max m, sum l, output O / l) of disjoint key ranges i,
//   out = sum_i 2^(m_i - M) l_i O_i / sum_i 2^(m_i - M) l_i,  M = max m_i,
// so the prefix and each sequence's own keys are attended to apart, each cut
// into page runs, and folded at the end.  Three launches: the query rows are
// quantized (q_quant.hip), the page runs attended to, the states folded.
//
// The work is a list of segments: first the prefix once for every eight
// consecutive tokens of the batch (48 rows of a KV head: three full 16-row
// tiles, whichever sequences they belong to), then each sequence's own pages
// for its tokens (nine or ten tokens: two segments).  Laid end to end, with a
// fixed cost ahead of each segment's pages, they form one axis that is cut
// into equal parts, one per work-group, so a work-group takes one or more
// pieces of consecutive segments and all end together: a prefix of 2,000 pages
// beside 200 sequences of two pages keeps the chip as busy as one of either
// kind alone.  Every work-group derives the same cut from the lengths on the
// device, so a captured call follows them.
//
// Inside a piece the kernel is the decode split kernel's: per KV head two
// waves (head dim 256: the half-heads of a pair) over rings of LDS slots
// filled by direct-to-LDS loads, see decode_chunk.h and decode.hip.  The device
// code of axis and pieces is in decode_pieces.h.
#include "decode_pieces.h"

namespace k8v4 {
namespace {

template <int NT, int HKV, int NWH, bool PH>
__global__ __attribute__((amdgpu_flat_work_group_size(64 * HKV * NWH, 64 * HKV * NWH),
                          amdgpu_waves_per_eu(SplitConfig<128, NT, HKV, NWH, PH>::OCC,
                                              SplitConfig<128, NT, HKV, NWH, PH>::OCC)))
void shared_split_kernel(PieceArgs args) {
  __shared__ __attribute__((aligned(16))) char lds[SplitConfig<128, NT, HKV, NWH, PH>::LDS_BYTES];
  const int wg = static_cast<int>(blockIdx.x);
  walk_pieces(args, wg, [&](const PieceArgs &a, int tid, int seg, int s0, int s1) {
    attend_piece<NT, HKV, NWH, PH, true>(a, lds, tid, wg, seg, s0, s1);
  });
}


// The many-rows form of the whole launch: the prefix's segments (KV heads x row
// blocks) by wide_piece, the sequences' own by attend_piece on the same axis.
template <int D, int HKV, int NT>
__global__ __attribute__((amdgpu_flat_work_group_size(512, 512), amdgpu_waves_per_eu(2, 2)))
void shared_wide_kernel(PieceArgs args) {
  constexpr bool PH = D == 256;
  constexpr int WAVE_HEADS = PH ? 2 * HKV : HKV, NWH = WAVE_HEADS == 8 ? 1 : 2;
  constexpr int OWN_LDS = SplitConfig<128, NT, WAVE_HEADS, NWH, PH>::LDS_BYTES;
  __shared__ __attribute__((aligned(16))) char lds[OWN_LDS > Wide<D>::LDS_BYTES ? OWN_LDS : Wide<D>::LDS_BYTES];
  const int wg = static_cast<int>(blockIdx.x);
  walk_pieces(args, wg, [&](const PieceArgs &a, int tid, int seg, int s0, int s1) {
    if (seg < a.groups)
      wide_piece<D, HKV>(a, lds, tid, wg, seg, s0, s1);
    else
      attend_piece<NT, WAVE_HEADS, NWH, PH, false, kWideWaves>(a, lds, tid, wg, seg, s0, s1);
  });
}


template <int HKV, int NWH, bool PH>
void launch_split(const PieceArgs &a, int tiles, hipStream_t s) {
  const dim3 grid(a.grid), block(64 * HKV * NWH);
  if (tiles == 1)
    shared_split_kernel<1, HKV, NWH, PH><<<grid, block, 0, s>>>(a);
  else if (tiles == 2)
    shared_split_kernel<2, HKV, NWH, PH><<<grid, block, 0, s>>>(a);
  else
    shared_split_kernel<3, HKV, NWH, PH><<<grid, block, 0, s>>>(a);
}

template <int D, int HKV>
void launch_wide(const PieceArgs &a, int tiles, hipStream_t s) {
  const dim3 grid(a.grid), block(64 * kWideWaves);
  if (tiles == 1)
    shared_wide_kernel<D, HKV, 1><<<grid, block, 0, s>>>(a);
  else if (tiles == 2)
    shared_wide_kernel<D, HKV, 2><<<grid, block, 0, s>>>(a);
  else
    shared_wide_kernel<D, HKV, 3><<<grid, block, 0, s>>>(a);
}

// Which form serves a prefix of `pages` pages for `rows` query rows of a KV head,
// of `batch` sequences: the many-rows kernel, or the one that takes eight tokens
// at a time.  Up to half a block of rows (a quarter at head dim 256) the former is
// the shorter chain unless the prefix is long beside them; beyond, it pays once the
// pages that each group of eight tokens would read again outweigh the waves it
// leaves idle, and with two 128-dim heads also what it loses on each sequence's own
// pages, which it serves with half as many work-groups.  Measured on both sides of
// every line, us, eight tokens at a time / many rows, at so many pages (sequences x
// query tokens, 100 tokens of each sequence's own):
//   D 128, 4 heads   8 x 1   256: 23.8 / 23.5   384: 25.9 / 26.6   625: 29.3 / 33.9
//                    5 x 7   192: 30.4 / 29.9   256: 32.4 / 31.3   384: 36.7 / 34.9
//                    64 x 1  128: 35.0 / 35.7   192: 38.3 / 37.9   256: 41.8 / 40.1
//                    128 x 1  32: 34.5 / 36.7    64: 38.2 / 39.4    96: 42.2 / 41.6
//                    48 x 4    8: 28.9 / 29.1    16: 31.3 / 29.7    32: 35.9 / 32.4
//   D 128, 2 heads   8 x 1   384: 22.7 / 21.5   625: 24.6 / 24.6
//                    64 x 1  256: 34.2 / 34.9   384: 37.9 / 37.7   625: 44.7 / 40.0
//                    32 x 4  192: 35.9 / 37.9   256: 39.7 / 39.0   384: 45.1 / 42.3
//                    256 x 1 192: 54.7 / 56.4   256: 63.0 / 61.2   384: 78.7 / 69.3
//                    64 x 4   96: 37.2 / 37.9   128: 41.1 / 39.6   192: 48.4 / 43.4
//   D 256, 2 heads   8 x 1   256: 24.3 / 23.8   384: 26.1 / 26.0   625: 29.1 / 30.3
//                    24 x 1  256: 31.5 / 33.5   384: 35.4 / 35.4   625: 42.1 / 39.4
//                    64 x 1  192: 41.3 / 43.4   256: 46.0 / 45.8
//                    128 x 1  64: 42.1 / 43.9    96: 46.7 / 47.1   128: 51.5 / 49.2
//                    64 x 4   32: 37.9 / 38.2    64: 47.5 / 43.4
//   D 256, 4 heads   8 x 1   256: 29.8 / 27.9   384: 31.6 / 32.4   625: 34.9 / 40.8
//                    5 x 7     8: 24.5 / 29.2   128: 35.2 / 37.3   192: 42.5 / 39.0
//                    64 x 4    8: 42.8 / 37.9    64: 73.1 / 53.9
// Over 1,392 shapes (48 to 2,304 rows, 8 to 2,048 pages, 1 to 10 query tokens) the
// form chosen is 0.2 % slower than the faster one on average and over 10 % slower at
// eight of them (five sequences of seven tokens over a few pages, four 256-dim heads:
// 19 %).  With 1,000 own tokens the lines lie at about the same pages (0.7 % on
// average; two sequences over long prefixes, four 256-dim heads: up to 32 %).
bool wide_pays(int64_t batch, int64_t rows, int64_t pages, int hkv, int head_dim) {
  if (rows <= (head_dim == 128 ? 192 : 96)) return rows >= (head_dim == 128 ? 144 : 84) || pages <= 8 * rows;
  if (head_dim == 256) return hkv == 4 || pages >= 384 || rows * pages >= 80000;
  if (hkv == 4) return 3 * pages + rows >= 960;
  return 4 * (pages - batch) + rows >= 1900;
}

// The form of a call (false where nothing is shared).
bool takes_many_rows(int64_t batch, int q_len, int hkv, int head_dim, int64_t prefix_pages) {
  return prefix_pages > 0 && wide_pays(batch, batch * q_len * kGqa, prefix_pages, hkv, head_dim);
}

int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

// What a call keeps in its workspace in one of the two forms: the quantized
// query rows, their scales, the states of the prefix's pieces and the others'.
struct SharedShape {
  int64_t tokens, groups, per_seq, head_rows, grid;
  int64_t blocks;  // row blocks of the many-rows form (0: eight tokens at a time)
  int prefix_rows, own_rows;
  int64_t prefix_bytes, own_bytes;
  int64_t q_bytes, scale_bytes, prefix_state_bytes, own_state_bytes;
  int64_t bytes() const { return q_bytes + scale_bytes + prefix_state_bytes + own_state_bytes; }
};
SharedShape shape_of(bool wide, int64_t batch, int q_len, int hkv, int head_dim) {
  SharedShape s;
  s.tokens = batch * q_len;
  s.per_seq = (q_len + kGroup - 1) / kGroup;
  const int64_t rows = s.tokens * kGqa, state = 2 * head_dim + 8;
  const int block_rows = head_dim == 128 ? Wide<128>::ROWS : Wide<256>::ROWS;
  s.blocks = wide ? (rows + block_rows - 1) / block_rows : 0;
  // One work-group per CU, two of the half-sized ones of two 128-dim heads.
  s.grid = static_cast<int64_t>(device_cus()) * (hkv == 2 && head_dim == 128 && !wide ? 2 : 1);
  s.own_rows = (q_len < kGroup ? q_len : kGroup) * kGqa;
  s.own_bytes = hkv * s.own_rows * state;
  if (wide) {
    s.groups = hkv * s.blocks;
    s.prefix_rows = block_rows;
    s.prefix_bytes = block_rows * state;
  } else {
    s.groups = (s.tokens + kGroup - 1) / kGroup;
    s.prefix_rows = static_cast<int>(s.tokens < kGroup ? s.tokens : kGroup) * kGqa;
    s.prefix_bytes = hkv * s.prefix_rows * state;
  }
  // A last segment's tiles, or a last block's rows, read rows behind the last token's.
  s.head_rows = s.blocks * block_rows > rows + 3 * 16 ? s.blocks * block_rows : rows + 3 * 16;
  s.q_bytes = round256(hkv * s.head_rows * head_dim);
  s.scale_bytes = round256(hkv * s.head_rows * 4);
  s.prefix_state_bytes = (s.grid + s.groups) * s.prefix_bytes;
  s.own_state_bytes = (s.grid + batch * s.per_seq) * s.own_bytes;
  return s;
}

constexpr int64_t kMaxBatch = int64_t(1) << 20;
constexpr int64_t kMaxPrefixPages = int64_t(1) << 24;

bool valid_shape(int64_t batch, int q_len, int hkv, int head_dim) {
  return batch >= 1 && batch <= kMaxBatch && q_len >= 1 && q_len <= kPage / kGqa && supported_heads(hkv) &&
         supported_dim(head_dim);
}

}  // namespace

int64_t shared_wait_timeouts() {
  int n = 0;
  const hipError_t e = hipMemcpyFromSymbol(&n, HIP_SYMBOL(g_pair_wait_timeouts), sizeof(n));
  if (e != hipSuccess) {
    set_error("k8v4_decode_fault_count: %s", hipGetErrorString(e));
    return -1;
  }
  return n;
}

}  // namespace k8v4

extern "C" int k8v4_attn_shared_many_rows(int64_t batch, int q_len, int hkv, int head_dim, int64_t prefix_len) {
  using namespace k8v4;
  if (!valid_shape(batch, q_len, hkv, head_dim) || prefix_len < 0 || prefix_len / kPage > kMaxPrefixPages) return -1;
  return takes_many_rows(batch, q_len, hkv, head_dim, prefix_len / kPage) ? 1 : 0;
}

extern "C" int64_t k8v4_attn_shared_workspace_bytes(int64_t batch, int q_len, int hkv, int head_dim) {
  using namespace k8v4;
  if (!valid_shape(batch, q_len, hkv, head_dim)) return -1;
  // Either form, whatever the prefix.
  const int64_t narrow = shape_of(false, batch, q_len, hkv, head_dim).bytes();
  const int64_t wide = shape_of(true, batch, q_len, hkv, head_dim).bytes();
  return narrow > wide ? narrow : wide;
}

extern "C" int k8v4_attn_shared(const void *q, int q_dtype, int64_t q_tok_stride, const int8_t *k_cache,
                                const float *k_scale, const uint8_t *v_cache, const float *v_scale,
                                const float *v_zero, int64_t num_pages, int64_t k_page_stride,
                                int64_t ks_page_stride, int64_t v_page_stride, int64_t vs_page_stride,
                                int64_t vz_page_stride, const int32_t *prefix_table, int64_t prefix_width,
                                int64_t prefix_len, const int32_t *block_table, int64_t bt_stride,
                                int64_t table_width, int pages_per_block, const int32_t *seq_lens, int64_t batch,
                                int q_len, int hkv, int head_dim, void *out, int out_dtype, int64_t out_tok_stride,
                                void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace k8v4;
  clear_error();
  K8V4_REQUIRE(supported_heads(hkv), "unsupported per-GPU KV head count %d (this library serves 2 or 4)", hkv);
  K8V4_REQUIRE(supported_dim(head_dim), "unsupported head dim %d (this library serves 128 or 256)", head_dim);
  K8V4_REQUIRE(q_len >= 1 && q_len <= kPage / kGqa, "q_len*GQA exceeds BM (q_len=%d)", q_len);
  K8V4_REQUIRE(pages_per_block >= 1, "pages_per_block");
  K8V4_REQUIRE(num_pages >= 1 && num_pages <= INT32_MAX, "num_pages must be 1 .. 2^31 - 1");
  K8V4_REQUIRE(batch >= 1 && batch <= kMaxBatch, "empty or too large batch");
  K8V4_REQUIRE(table_width >= 1 && table_width <= (int64_t(1) << 24) / pages_per_block, "block_table width");
  K8V4_REQUIRE(prefix_len >= 0, "negative prefix length");
  const int64_t prefix_pages = prefix_len / kPage;  // whole pages are shared, a part of one is each sequence's own
  K8V4_REQUIRE(prefix_pages <= kMaxPrefixPages, "prefix too long");
  K8V4_REQUIRE(prefix_pages == 0 || prefix_width >= (prefix_pages + pages_per_block - 1) / pages_per_block,
               "prefix_table has %lld entries, the prefix of %lld tokens needs %lld",
               static_cast<long long>(prefix_width), static_cast<long long>(prefix_len),
               static_cast<long long>((prefix_pages + pages_per_block - 1) / pages_per_block));
  K8V4_REQUIRE(q_dtype == K8V4_F16 || q_dtype == K8V4_BF16, "q dtype must be fp16 or bf16");
  K8V4_REQUIRE(out_dtype == K8V4_F16 || out_dtype == K8V4_BF16 || out_dtype == K8V4_F32,
               "out dtype must be fp16, bf16 or fp32");
  K8V4_REQUIRE(q && k_cache && k_scale && v_cache && v_scale && v_zero && block_table && seq_lens && out && workspace &&
                   (prefix_table || prefix_pages == 0),
               "null pointer");
  const auto aligned = [](const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  K8V4_REQUIRE(aligned(q, 16) && q_tok_stride % 8 == 0,
               "q must be 16-byte aligned with a token stride that is a multiple of 8 elements");
  const int64_t row = static_cast<int64_t>(hkv) * kGqa * head_dim;
  K8V4_REQUIRE(q_tok_stride >= row, "q token stride shorter than HQ*D");
  K8V4_REQUIRE(out_tok_stride >= row, "out token stride shorter than HQ*D");
  K8V4_REQUIRE(aligned(out, out_dtype == K8V4_F32 ? 4 : 2), "out misaligned");
  K8V4_REQUIRE(bt_stride >= table_width, "block_table row stride shorter than its width");
  K8V4_REQUIRE(aligned(block_table, 4) && aligned(prefix_table, 4) && aligned(seq_lens, 4), "index arrays misaligned");
  K8V4_REQUIRE(aligned(k_cache, 16) && k_page_stride % 16 == 0, "k_cache must keep 16-byte aligned rows");
  K8V4_REQUIRE(aligned(v_cache, 4) && v_page_stride % 4 == 0, "v_cache must keep 4-byte aligned rows");
  K8V4_REQUIRE(aligned(k_scale, 8) && aligned(v_scale, 8) && aligned(v_zero, 8) && ks_page_stride % 8 == 0 &&
                   vs_page_stride % 8 == 0 && vz_page_stride % 8 == 0,
               "scale planes must be 8-byte aligned");
  for (const int64_t stride : {k_page_stride, ks_page_stride, v_page_stride, vs_page_stride, vz_page_stride})
    K8V4_REQUIRE(stride >= 0 && stride < (int64_t(1) << 31), "cache page strides must be 0 .. 2^31 - 1 bytes");
  K8V4_REQUIRE(aligned(workspace, 16), "workspace must be 16-byte aligned");

  const int64_t need = k8v4_attn_shared_workspace_bytes(batch, q_len, hkv, head_dim);
  if (workspace_bytes < need) {
    set_error("shared-prefix workspace holds %lld bytes, the batch needs %lld", static_cast<long long>(workspace_bytes),
              static_cast<long long>(need));
    return K8V4_ERR_WORKSPACE;
  }
  const bool wide = takes_many_rows(batch, q_len, hkv, head_dim, prefix_pages);
  const SharedShape sh = shape_of(wide, batch, q_len, hkv, head_dim);
  const int64_t table_pages = table_width * pages_per_block;
  const int64_t groups = prefix_pages ? sh.groups : 0;
  // The axis has at most this many units; a work-group's end may pass it by a
  // work-group's share.
  const int64_t units = groups * (prefix_pages + kPieceCost) +
                        batch * sh.per_seq * ((table_pages > prefix_pages ? table_pages - prefix_pages : 0) + kPieceCost);
  K8V4_REQUIRE(units < (int64_t(1) << 30), "batch too large for one call");

  PieceArgs a;
  char *ws = static_cast<char *>(workspace);
  int8_t *q8 = reinterpret_cast<int8_t *>(ws);
  float *scales = reinterpret_cast<float *>(ws + sh.q_bytes);
  a.q8 = q8;
  a.q8_scale = scales;
  a.head_rows = sh.head_rows;
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
  {
    const int64_t dkv = reinterpret_cast<intptr_t>(v_scale) - reinterpret_cast<intptr_t>(k_scale);
    const int64_t dvz = reinterpret_cast<intptr_t>(v_zero) - reinterpret_cast<intptr_t>(v_scale);
    const int64_t lim = int64_t(1) << 30;
    a.planes_fast = ks_page_stride == vs_page_stride && vs_page_stride == vz_page_stride && dkv > -lim &&
                    dkv < lim && dvz > -lim && dvz < lim;
    a.d_kv = a.planes_fast ? dkv : 0;
    a.d_vz = a.planes_fast ? dvz : 0;
  }
  a.prefix_table = prefix_table;
  a.prefix_pages = static_cast<int>(prefix_pages);
  a.block_table = block_table;
  a.bt_stride = bt_stride;
  a.table_pages = static_cast<int>(table_pages);
  a.ppb = pages_per_block;
  a.seq_lens = seq_lens;
  a.batch = static_cast<int>(batch);
  a.q_len = q_len;
  a.hkv = hkv;
  a.tokens = static_cast<int>(sh.tokens);
  a.groups = static_cast<int>(groups);
  a.per_seq = static_cast<int>(sh.per_seq);
  a.wide_blocks = static_cast<int>(sh.blocks);
  a.grid = static_cast<int>(sh.grid);
  a.ws = ws + sh.q_bytes + sh.scale_bytes;
  a.own_ws = a.ws + sh.prefix_state_bytes;
  a.prefix_rows = sh.prefix_rows;
  a.own_rows = sh.own_rows;
  a.prefix_bytes = sh.prefix_bytes;
  a.own_bytes = sh.own_bytes;
  a.out = out;
  a.out_dtype = out_dtype;
  a.out_tok_stride = out_tok_stride;
  // The merge's column slices and threads, as for the decode merge: the fewest
  // with which one round of loads covers a row's pieces on average.
  int tpu = 256;
  {
    const int vpr_max = head_dim / 8;
    const int64_t avg = groups ? (sh.grid + groups - 1) / groups + 1 : (sh.grid + batch - 1) / batch;
    int cs = vpr_max / 8;
    bool found = false;
    for (int threads : {64, 128, 256}) {
      for (int c = 1; vpr_max / c >= 8 && !found; c *= 2) {
        const int spi = threads / (vpr_max / c);
        if ((avg + spi - 1) / spi <= kMergeMU) {
          cs = c;
          tpu = threads;
          found = true;
        }
      }
      if (found) break;
    }
    a.merge_cs = cs;
  }
  const int64_t merge_units = sh.tokens * kGqa * hkv * a.merge_cs;
  K8V4_REQUIRE(merge_units <= INT32_MAX / 2, "batch too large for one merge launch");

  auto s = static_cast<hipStream_t>(stream);
  int rc = q_rows_launch(q, q_dtype == K8V4_BF16, q_tok_stride, sh.tokens, hkv, head_dim, sh.head_rows, q8, scales, s);
  if (rc) return rc;
  const int widest = groups && !sh.blocks && sh.prefix_rows > sh.own_rows ? sh.prefix_rows : sh.own_rows;
  const int tiles = (widest + 15) / 16;
  if (sh.blocks) {
    if (head_dim == 256) {
      if (hkv == 4)
        launch_wide<256, 4>(a, tiles, s);
      else
        launch_wide<256, 2>(a, tiles, s);
    } else {
      if (hkv == 4)
        launch_wide<128, 4>(a, tiles, s);
      else
        launch_wide<128, 2>(a, tiles, s);
    }
  } else if (head_dim == 256) {
    if (hkv == 4)
      launch_split<8, 1, true>(a, tiles, s);
    else
      launch_split<4, 2, true>(a, tiles, s);
  } else {
    if (hkv == 4)
      launch_split<4, 2, false>(a, tiles, s);
    else
      launch_split<2, 2, false>(a, tiles, s);
  }
  rc = launch_status("k8v4_attn_shared split");
  if (rc) return rc;
  const dim3 mgrid(static_cast<unsigned>(merge_units));
  if (head_dim == 128) {
    if (tpu == 64)
      pieces_merge_kernel<128, 64><<<mgrid, dim3(64), 0, s>>>(a);
    else if (tpu == 128)
      pieces_merge_kernel<128, 128><<<mgrid, dim3(128), 0, s>>>(a);
    else
      pieces_merge_kernel<128, 256><<<mgrid, dim3(256), 0, s>>>(a);
  } else {
    if (tpu == 64)
      pieces_merge_kernel<256, 64><<<mgrid, dim3(64), 0, s>>>(a);
    else if (tpu == 128)
      pieces_merge_kernel<256, 128><<<mgrid, dim3(128), 0, s>>>(a);
    else
      pieces_merge_kernel<256, 256><<<mgrid, dim3(256), 0, s>>>(a);
  }
  return launch_status("k8v4_attn_shared merge");
}
