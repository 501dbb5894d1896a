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
// The work is cut as in decode_shared.hip, with no prefix: a sequence's segments
// are its runs of eight nodes (48 rows of a KV head), each over all its pages.
// Three launches: the query rows are quantized, the page runs attended to, their
// states folded.
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
  const int wg = static_cast<int>(blockIdx.x);
  walk_pieces<true>(args, wg, [&](const PieceArgs &a, int tid, int seg, int s0, int s1) {
    attend_piece<NT, HKV, NWH, PH, false, HKV * NWH, true>(a, lds, tid, wg, seg, s0, s1);
  });
}

// Many rows of one KV head: wide_piece in decode_pieces.h, TILES row tiles a wave.
template <int D, int HKV, int TILES>
__global__ __attribute__((amdgpu_flat_work_group_size(512, 512), amdgpu_waves_per_eu(2, 2)))
void tree_wide_kernel(PieceArgs args) {
  using W = Wide<D, TILES>;
  static_assert(W::LDS_BYTES + kWideWordBytes <= 163840, "no room for the mask words");
  __shared__ __attribute__((aligned(16))) char lds[W::LDS_BYTES + kWideWordBytes];
  const int wg = static_cast<int>(blockIdx.x);
  walk_pieces<true>(args, wg, [&](const PieceArgs &a, int tid, int seg, int s0, int s1) {
    wide_piece<D, HKV, TILES, true>(a, lds, tid, wg, seg, s0, s1);
  });
}

template <int D, int HKV>
void launch_wide(const PieceArgs &a, int tiles, hipStream_t s) {
  const dim3 grid(a.grid), block(64 * kWideWaves);
  if (tiles == 1)
    tree_wide_kernel<D, HKV, 1><<<grid, block, 0, s>>>(a);
  else if (D == 256 || tiles == 2)
    tree_wide_kernel<D, HKV, 2><<<grid, block, 0, s>>>(a);
  else
    tree_wide_kernel<D, HKV, D == 256 ? 2 : 3><<<grid, block, 0, s>>>(a);
}

template <int HKV, int NWH, bool PH>
void launch_split(const PieceArgs &a, int tiles, hipStream_t s) {
  const dim3 grid(a.grid), block(64 * HKV * NWH);
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
  int64_t tokens, per_seq, head_rows, grid;
  int64_t blocks;  // row blocks of a KV head in the wide form (0: eight nodes at a time)
  int tiles;       // row tiles of a wave
  int own_rows;
  int64_t own_bytes;
  int64_t q_bytes, scale_bytes, state_bytes;
  int64_t bytes() const { return q_bytes + scale_bytes + state_bytes; }
};
TreeShape shape_of(bool wide, int64_t batch, int nodes, int hkv, int head_dim) {
  TreeShape s;
  s.tokens = batch * nodes;
  const int64_t rows = static_cast<int64_t>(nodes) * kGqa, state = 2 * head_dim + 8;
  if (wide) {
    const int most = head_dim == 128 ? Wide<128>::NT : Wide<256>::NT, tile_rows = kWideWaves * 16;
    const int64_t tiles = (rows + tile_rows - 1) / tile_rows;
    s.blocks = (tiles + most - 1) / most;
    s.tiles = static_cast<int>((tiles + s.blocks - 1) / s.blocks);
    s.own_rows = tile_rows * s.tiles;
    s.per_seq = hkv * s.blocks;
    s.own_bytes = s.own_rows * state;
    s.grid = device_cus();
    s.head_rows = s.tokens * kGqa + s.own_rows;  // a last block's tiles read rows behind the last token's
  } else {
    s.blocks = 0;
    s.per_seq = (nodes + kGroup - 1) / kGroup;
    s.own_rows = (nodes < kGroup ? nodes : kGroup) * kGqa;
    s.tiles = (s.own_rows + 15) / 16;
    s.own_bytes = hkv * s.own_rows * state;
    // One work-group per CU, two of the half-sized ones of two 128-dim heads.
    s.grid = static_cast<int64_t>(device_cus()) * (hkv == 2 && head_dim == 128 ? 2 : 1);
    s.head_rows = s.tokens * kGqa + 3 * 16;
  }
  s.q_bytes = round256(hkv * s.head_rows * head_dim);
  s.scale_bytes = round256(hkv * s.head_rows * 4);
  s.state_bytes = (s.grid + batch * s.per_seq) * s.own_bytes;
  return s;
}

// Which form serves trees of so many nodes.
bool takes_wide(int nodes) { return nodes > kGroup; }

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
  return shape_of(takes_wide(nodes), batch, nodes, hkv, head_dim).bytes();
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
  const TreeShape sh = shape_of(takes_wide(nodes), batch, nodes, hkv, head_dim);
  const int64_t table_pages = table_width * pages_per_block;
  K8V4_REQUIRE(batch * sh.per_seq * (table_pages + kPieceCost) < (int64_t(1) << 30), "batch too large for one call");

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
  a.per_seq = static_cast<int>(sh.per_seq);
  a.wide_blocks = static_cast<int>(sh.blocks);
  a.grid = static_cast<int>(sh.grid);
  a.ws = a.own_ws = ws + sh.q_bytes + sh.scale_bytes;
  a.own_rows = sh.own_rows;
  a.own_bytes = sh.own_bytes;
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
    const int64_t segments = batch * sh.per_seq;
    const int64_t avg = (sh.grid + segments - 1) / segments;
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
