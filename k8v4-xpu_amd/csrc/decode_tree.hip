// Paged decode attention of drafted trees: the query tokens of a sequence are the
// nodes of a tree of drafted tokens, stored behind its context, and each sees the
// context and, of the tree, the nodes its mask holds (its own branch).
//
// Node j of sequence b is the token at position len_b - nodes + j.  With context
// c = len_b - nodes, a query row of node j attends to the keys t < c and to the
// keys c + i whose bit i is set in mask[b][j], by softmax attention as in
// k8v4_attn_batch (int8-quantized query rows, exact integer dot products, V as
// (nibble - zero) * scale); a row that sees no key gives zeros.
//
// The work is cut as in decode_shared.hip, with no prefix: the sequences' pages make
// the axis, and several work-groups share a part of it, either one for every eight
// nodes (48 rows of all KV heads) or one for every KV head and block of its rows.
// Three launches: the query rows are quantized (not where the second form does that
// itself), the page runs attended to, their states folded.
//
// Roundings to fewer than 32 bits are the batch op's (probabilities, V scales or
// dequantized V and a page run's output in fp16, the query int8): with them both
// products run on the matrix cores at 16 and 8 bits.  Sums, maxima and the folding
// are fp32.
#include "decode_pieces.h"

namespace k8v4 {
namespace {

constexpr int kMaxNodes = 64;  // bits of a mask word

template <int NT, int HKV, int NWH, bool PH>
__global__ __attribute__((amdgpu_flat_work_group_size(64 * HKV * NWH, 64 * HKV * NWH),
                          amdgpu_waves_per_eu(SplitConfig<128, NT, HKV, NWH, PH>::OCC,
                                              SplitConfig<128, NT, HKV, NWH, PH>::OCC)))
void tree_split_kernel(PieceArgs args) {
  using CFG = SplitConfig<128, NT, HKV, NWH, PH>;
  static_assert(CFG::LDS_BYTES + kTreeWordBytes <= CFG::LDS_MAX, "no room for the mask words");
  __shared__ __attribute__((aligned(16))) char lds[CFG::LDS_BYTES + kTreeWordBytes];
  const int wg = tree_place(args).part;
  walk_pieces(args, wg, [&](const PieceArgs &a, int tid, int seg, int s0, int s1) {
    attend_piece<NT, HKV, NWH, PH, false, HKV * NWH, true>(a, lds, tid, wg, seg, s0, s1);
  });
}

// Work-groups of the wide form on a CU.  With one 128-dim row tile a wave a phase is
// short and mostly latency; two work-groups fill each other's gaps (8 nodes over four
// times 100,000 tokens 98 us, with one work-group of four ring slots 126, of eight
// slots 126).
constexpr int wide_groups(int head_dim, int tiles) { return head_dim == 128 && tiles == 1 ? 2 : 1; }

// Many rows of one KV head: wide_piece in decode_pieces.h, TILES row tiles a wave.
// Bound by issue: 64 nodes over four times 100,000 tokens (4 KV heads, D 128) 271 us,
// 1,045 TFLOP/s of products (two thirds of them fp16's share of the time); 16 nodes,
// where unpacking a page for all waves weighs more, 133 us.
template <int D, int HKV, int TILES>
__global__ __attribute__((amdgpu_flat_work_group_size(512, 512),
                          amdgpu_waves_per_eu(2 * wide_groups(D, TILES), 2 * wide_groups(D, TILES))))
void tree_wide_kernel(PieceArgs args) {
  constexpr int GROUPS = wide_groups(D, TILES), RING = GROUPS == 2 ? 3 : Wide<D>::SLOTS;
  using W = Wide<D, TILES, RING>;
  static_assert(W::LDS_BYTES + kWideWordBytes <= 163840 / GROUPS, "no room for the mask words");
  __shared__ __attribute__((aligned(16))) char lds[W::LDS_BYTES + kWideWordBytes];
  const int wg = tree_place(args).part;
  walk_pieces(args, wg, [&](const PieceArgs &a, int tid, int seg, int s0, int s1) {
    wide_piece<D, HKV, TILES, true, RING>(a, lds, tid, wg, seg, s0, s1);
  });
}

template <int D, int HKV>
void launch_wide(const PieceArgs &a, int tiles, hipStream_t s) {
  const dim3 grid(a.grid * a.shares), block(64 * kWideWaves);
  if (tiles == 1)
    tree_wide_kernel<D, HKV, 1><<<grid, block, 0, s>>>(a);
  else if (D == 256 || tiles == 2)
    tree_wide_kernel<D, HKV, 2><<<grid, block, 0, s>>>(a);
  else
    tree_wide_kernel<D, HKV, D == 256 ? 2 : 3><<<grid, block, 0, s>>>(a);
}

template <int HKV, int NWH, bool PH>
void launch_split(const PieceArgs &a, int tiles, hipStream_t s) {
  const dim3 grid(a.grid * a.shares), block(64 * HKV * NWH);
  if (tiles == 1)
    tree_split_kernel<1, HKV, NWH, PH><<<grid, block, 0, s>>>(a);
  else if (tiles == 2)
    tree_split_kernel<2, HKV, NWH, PH><<<grid, block, 0, s>>>(a);
  else
    tree_split_kernel<3, HKV, NWH, PH><<<grid, block, 0, s>>>(a);
}

int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

// What a call keeps in its workspace: the quantized query rows, their scales and
// the states of the pieces.
struct TreeShape {
  int64_t tokens, head_rows;
  int64_t grid;    // parts of the axis
  int shares;      // work-groups of a part
  int64_t blocks;  // row blocks of a KV head in the wide form (0: eight nodes at a time)
  int tiles;       // row tiles of a wave
  int own_rows;
  int64_t share_bytes;
  int64_t q_bytes, scale_bytes, state_bytes;
  int64_t bytes() const { return q_bytes + scale_bytes + state_bytes; }
};
TreeShape shape_of(bool wide, int64_t batch, int nodes, int hkv, int head_dim) {
  TreeShape s;
  s.tokens = batch * nodes;
  const int64_t rows = static_cast<int64_t>(nodes) * kGqa, state = 2 * head_dim + 8;
  int64_t groups = device_cus();  // work-groups: one per CU
  if (wide) {
    const int most = head_dim == 128 ? Wide<128>::NT : Wide<256>::NT, tile_rows = kWideWaves * 16;
    const int64_t tiles = (rows + tile_rows - 1) / tile_rows;
    s.blocks = (tiles + most - 1) / most;
    s.tiles = static_cast<int>((tiles + s.blocks - 1) / s.blocks);
    s.own_rows = tile_rows * s.tiles;
    s.shares = static_cast<int>(hkv * s.blocks);
    groups *= wide_groups(head_dim, s.tiles);
    s.share_bytes = s.own_rows * state;
    // A last block's tiles read rows behind the last token's.
    s.head_rows = tree_quantizes(head_dim, s.tiles) ? 0 : s.tokens * kGqa + s.own_rows;
  } else {
    if (hkv == 2 && head_dim == 128) groups *= 2;  // half-sized ones
    s.blocks = 0;
    s.own_rows = (nodes < kGroup ? nodes : kGroup) * kGqa;
    s.tiles = (s.own_rows + 15) / 16;
    s.shares = (nodes + kGroup - 1) / kGroup;
    s.share_bytes = hkv * s.own_rows * state;
    s.head_rows = s.tokens * kGqa + 3 * 16;
  }
  const int64_t parts = groups / (8 * s.shares) * 8;
  s.grid = parts > 8 ? parts : 8;
  s.q_bytes = round256(hkv * s.head_rows * head_dim);
  s.scale_bytes = round256(hkv * s.head_rows * 4);
  s.state_bytes = (s.grid + batch) * s.shares * s.share_bytes;
  return s;
}

// Which form serves trees of so many nodes over tables of so many pages in all (of
// the lengths the host knows no more: a table wider than its sequences need has the
// form of longer ones, with their costs): the wide form, or eight nodes at a time.  A
// wide page costs about as much for 1 as for 20 nodes (unpacked once for all rows, in
// phases that wait for each other), the other form's about the same for each run of
// eight; over a few pages the latter has the longer chain, but for the wide form's
// row blocks of two and three tiles a wave.  Measured, us, eight at a time / wide, at
// so many pages (4,000 tokens of one sequence to 100,000 of four):
//   D 128, 4 heads   4 nodes    63: 18.7 / 14.9   254: 19.8 / 20.2  1004: 27.8 / 29.1  6256: 68 / 93
//                    8          63: 21.1 / 15.9   504: 25.8 / 24.6  1004: 30.9 / 30.1  6256: 71 / 98
//                    16         63: 21.8 / 18.4  1004: 35.9 / 37.3  2004: 48.8 / 52.6  6256: 112 / 133
//                    17         63: 22.2 / 19.1  1008: 53.0 / 45.0                     6256: 159 / 138
//                    21         33: 21.4 / 18.4  1032: 46.1 / 40.9                     6256: 160 / 145
//                    26         63: 22.1 / 20.2   252: 30.7 / 29.1   504: 41.1 / 34.9  1004: 50.9 / 43.1
//                    32         63: 22.9 / 21.2   252: 32.0 / 29.8   504: 42.5 / 36.9
//                    42         63: 24.3 / 27.0   126: 29.2 / 27.0   252: 37.1 / 34.9
//                    64         63: 26.2 / 35.2   254: 40.7 / 45.0   504: 54.0 / 44.7  6256: 406 / 271
//   D 128, 2 heads   8          63: 19.0 / 15.4   504: 24.1 / 21.1  2004: 30.3 / 28.9  6256: 46 / 56
//                    21         63: 20.5 / 19.0  1008: 36.8 / 33.4                     6256: 88 / 77
//                    32         63: 20.8 / 21.0   126: 22.5 / 21.6   252: 26.2 / 25.9
//                    42         63: 22.7 / 23.3   126: 24.8 / 27.1   252: 27.2 / 27.3
//                    64        254: 30.8 / 37.1   504: 43.1 / 45.0   756: 55.8 / 53.9
//                             1004: 51.1 / 50.4  2004: 74.7 / 65.1
//   D 256, 2 heads   8          63: 21.5 / 18.2   504: 26.4 / 25.0  1004: 32.5 / 32.3  2004: 39.8 / 46.6
//                    16         63: 21.7 / 21.3  1004: 38.9 / 37.8  2004: 55.0 / 53.9
//                    21         63: 23.5 / 22.7  1008: 55.9 / 45.8                     6256: 190 / 140
//                    26        126: 26.7 / 27.1   252: 31.4 / 33.1   504: 40.9 / 38.3
//                    42        127: 29.2 / 35.6   254: 36.8 / 36.7   504: 49.2 / 44.7  2004: 126 / 79
//   D 256, 4 heads   8          63: 24.2 / 18.8   504: 33.2 / 32.1  1004: 42.5 / 46.8  2004: 56.8 / 75.1
//                    21         63: 28.3 / 23.7  1008: 88.4 / 70.9                     6256: 363 / 269
//                    26         63: 28.0 / 26.7
//                    42         63: 31.9 / 35.3   127: 39.9 / 36.6   504: 77.5 / 54.4  2004: 222 / 123
//                    50         63: 34.7 / 35.0   126: 44.6 / 43.6   252: 59.8 / 51.1
//                    64         63: 36.6 / 35.4   252: 61.1 / 52.9   504: 110 / 90.4
// The lines are simple, and next to them the slower form may be taken: by up to 4 % (4
// nodes at 254 pages, 16 at 1,004, 64 of two 128-dim heads from 384 to about 700), and
// by a tenth for about 42 nodes of four 256-dim heads over one sequence of 4,000 tokens.
bool takes_wide(int nodes, int64_t pages, int hkv, int head_dim) {
  if (nodes <= 16) return pages <= 64 * nodes;
  if (nodes <= 21 || (hkv == 4 && head_dim == 256)) return true;  // one row tile a wave, or half as much LDS a row
  if (head_dim == 128 && (nodes <= 32 || (nodes <= 42 && hkv == 4 && pages > 96))) return true;  // two
  return pages > 384;
}

constexpr int64_t kMaxBatch = int64_t(1) << 20;

bool valid_shape(int64_t batch, int nodes, int hkv, int head_dim) {
  return batch >= 1 && batch <= kMaxBatch && nodes >= 1 && nodes <= kMaxNodes && supported_heads(hkv) &&
         supported_dim(head_dim);
}

}  // namespace

int64_t tree_wait_timeouts() {
  int n = 0;
  const hipError_t e = hipMemcpyFromSymbol(&n, HIP_SYMBOL(g_pair_wait_timeouts), sizeof(n));
  if (e != hipSuccess) {
    set_error("k8v4_decode_fault_count: %s", hipGetErrorString(e));
    return -1;
  }
  return n;
}

}  // namespace k8v4

extern "C" int64_t k8v4_attn_tree_workspace_bytes(int64_t batch, int nodes, int hkv, int head_dim) {
  using namespace k8v4;
  if (!valid_shape(batch, nodes, hkv, head_dim)) return -1;
  // Either form, whatever the tables.
  const int64_t narrow = shape_of(false, batch, nodes, hkv, head_dim).bytes();
  const int64_t wide = shape_of(true, batch, nodes, hkv, head_dim).bytes();
  return narrow > wide ? narrow : wide;
}

extern "C" int k8v4_attn_tree(const void *q, int q_dtype, int64_t q_tok_stride, const int8_t *k_cache,
                              const float *k_scale, const uint8_t *v_cache, const float *v_scale, const float *v_zero,
                              int64_t num_pages, int64_t k_page_stride, int64_t ks_page_stride, int64_t v_page_stride,
                              int64_t vs_page_stride, int64_t vz_page_stride, const int32_t *block_table,
                              int64_t bt_stride, int64_t table_width, int pages_per_block, const int32_t *seq_lens,
                              const int64_t *tree_masks, int64_t mask_stride, int64_t batch, int nodes, int hkv,
                              int head_dim, void *out, int out_dtype, int64_t out_tok_stride, void *workspace,
                              int64_t workspace_bytes, void *stream) {
  using namespace k8v4;
  clear_error();
  K8V4_REQUIRE(supported_heads(hkv), "unsupported per-GPU KV head count %d (this library serves 2 or 4)", hkv);
  K8V4_REQUIRE(supported_dim(head_dim), "unsupported head dim %d (this library serves 128 or 256)", head_dim);
  K8V4_REQUIRE(nodes >= 1 && nodes <= kMaxNodes, "1 to %d nodes a tree, got %d", kMaxNodes, nodes);
  K8V4_REQUIRE(pages_per_block >= 1, "pages_per_block");
  K8V4_REQUIRE(num_pages >= 1 && num_pages <= INT32_MAX, "num_pages must be 1 .. 2^31 - 1");
  K8V4_REQUIRE(batch >= 1 && batch <= kMaxBatch, "empty or too large batch");
  K8V4_REQUIRE(table_width >= 1 && table_width <= (int64_t(1) << 24) / pages_per_block, "block_table width");
  K8V4_REQUIRE(q_dtype == K8V4_F16 || q_dtype == K8V4_BF16, "q dtype must be fp16 or bf16");
  K8V4_REQUIRE(out_dtype == K8V4_F16 || out_dtype == K8V4_BF16 || out_dtype == K8V4_F32,
               "out dtype must be fp16, bf16 or fp32");
  K8V4_REQUIRE(q && k_cache && k_scale && v_cache && v_scale && v_zero && block_table && seq_lens && tree_masks && out &&
                   workspace,
               "null pointer");
  const auto aligned = [](const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  K8V4_REQUIRE(aligned(q, 16) && q_tok_stride % 8 == 0,
               "q must be 16-byte aligned with a token stride that is a multiple of 8 elements");
  const int64_t row = static_cast<int64_t>(hkv) * kGqa * head_dim;
  K8V4_REQUIRE(q_tok_stride >= row, "q token stride shorter than HQ*D");
  K8V4_REQUIRE(out_tok_stride >= row, "out token stride shorter than HQ*D");
  K8V4_REQUIRE(aligned(out, out_dtype == K8V4_F32 ? 4 : 2), "out misaligned");
  K8V4_REQUIRE(bt_stride >= table_width || batch == 1, "block_table row stride shorter than its width");
  K8V4_REQUIRE(mask_stride >= nodes || mask_stride == 0, "tree_masks row stride shorter than the nodes");
  K8V4_REQUIRE(aligned(block_table, 4) && aligned(seq_lens, 4) && aligned(tree_masks, 8), "index arrays misaligned");
  K8V4_REQUIRE(aligned(k_cache, 16) && k_page_stride % 16 == 0, "k_cache must keep 16-byte aligned rows");
  K8V4_REQUIRE(aligned(v_cache, 4) && v_page_stride % 4 == 0, "v_cache must keep 4-byte aligned rows");
  K8V4_REQUIRE(aligned(k_scale, 8) && aligned(v_scale, 8) && aligned(v_zero, 8) && ks_page_stride % 8 == 0 &&
                   vs_page_stride % 8 == 0 && vz_page_stride % 8 == 0,
               "scale planes must be 8-byte aligned");
  for (const int64_t stride : {k_page_stride, ks_page_stride, v_page_stride, vs_page_stride, vz_page_stride})
    K8V4_REQUIRE(stride >= 0 && stride < (int64_t(1) << 31), "cache page strides must be 0 .. 2^31 - 1 bytes");
  K8V4_REQUIRE(aligned(workspace, 16), "workspace must be 16-byte aligned");

  const int64_t need = k8v4_attn_tree_workspace_bytes(batch, nodes, hkv, head_dim);
  if (workspace_bytes < need) {
    set_error("tree workspace holds %lld bytes, the batch needs %lld", static_cast<long long>(workspace_bytes),
              static_cast<long long>(need));
    return K8V4_ERR_WORKSPACE;
  }
  const int64_t table_pages = table_width * pages_per_block;
  const TreeShape sh = shape_of(takes_wide(nodes, batch * table_pages, hkv, head_dim), batch, nodes, hkv, head_dim);
  K8V4_REQUIRE(batch * (table_pages + kPieceCost) < (int64_t(1) << 30), "batch too large for one call");

  PieceArgs a = {};
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
  a.block_table = block_table;
  a.bt_stride = bt_stride;
  a.table_pages = static_cast<int>(table_pages);
  a.ppb = pages_per_block;
  a.seq_lens = seq_lens;
  a.batch = static_cast<int>(batch);
  a.q_len = nodes;
  a.hkv = hkv;
  a.tokens = static_cast<int>(sh.tokens);
  a.per_seq = 1;
  a.wide_blocks = static_cast<int>(sh.blocks);
  a.grid = static_cast<int>(sh.grid);
  a.ws = a.own_ws = ws + sh.q_bytes + sh.scale_bytes;
  a.own_rows = sh.own_rows;
  a.own_bytes = sh.shares * sh.share_bytes;
  a.q = static_cast<const uint16_t *>(q);
  a.q_bf16 = q_dtype == K8V4_BF16;
  a.q_tok_stride = q_tok_stride;
  a.shares = sh.shares;
  a.share_bytes = sh.share_bytes;
  a.out = out;
  a.out_dtype = out_dtype;
  a.out_tok_stride = out_tok_stride;
  a.tree_masks = tree_masks;
  a.mask_stride = mask_stride;
  // The merge's column slices and threads, as for the decode merge: the fewest
  // with which one round of loads covers a row's pieces on average.
  int tpu = 256;
  {
    const int vpr_max = head_dim / 8;
    const int64_t avg = (sh.grid + batch - 1) / batch;
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
  int rc = sh.head_rows == 0 ? K8V4_OK : q_rows_launch(q, q_dtype == K8V4_BF16, q_tok_stride, sh.tokens, hkv, head_dim, sh.head_rows, q8, scales, s);
  if (rc) return rc;
  const int tiles = sh.tiles;
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
  rc = launch_status("k8v4_attn_tree split");
  if (rc) return rc;
  const dim3 mgrid(static_cast<unsigned>(merge_units));
  if (head_dim == 128) {
    if (tpu == 64)
      pieces_merge_kernel<128, 64, true><<<mgrid, dim3(64), 0, s>>>(a);
    else if (tpu == 128)
      pieces_merge_kernel<128, 128, true><<<mgrid, dim3(128), 0, s>>>(a);
    else
      pieces_merge_kernel<128, 256, true><<<mgrid, dim3(256), 0, s>>>(a);
  } else {
    if (tpu == 64)
      pieces_merge_kernel<256, 64, true><<<mgrid, dim3(64), 0, s>>>(a);
    else if (tpu == 128)
      pieces_merge_kernel<256, 128, true><<<mgrid, dim3(128), 0, s>>>(a);
    else
      pieces_merge_kernel<256, 256, true><<<mgrid, dim3(256), 0, s>>>(a);
  }
  return launch_status("k8v4_attn_tree merge");
}
