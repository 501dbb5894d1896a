// The branch of a drafted tree that the target's tokens confirm: what follows the
// tree attention, the model's head and the choice (greedy or sampled) of the
// target's token after every node.  No counterpart in the reference.
//
// Sequence b's node 0 is its last token, node i > 0 a drafted token x_i that
// continues node parents[i] < i; t_i is the token the target chose after node i's
// branch.  From node 0 on the walk goes to the lowest child whose draft is the
// token chosen at the node, until there is none: a nodes are passed, and the token
// chosen at the last of them is new.  The tokens of a walk are the target's own
// choices, so they are distributed as the target's, however the drafts were made.
//
// One wave a sequence, a lane a node (64 at most): a step is a comparison in every
// lane and a ballot.  Bound by the launch: the nodes are 16 bytes each (2.2 us for one
// tree of 13, 3.7 for 256 trees of 64).
#include "k8v4_common.h"

namespace k8v4 {
namespace {

constexpr int kMaxNodes = 64;
constexpr int kSeqs = 4;  // sequences of a work-group

struct AcceptArgs {
  const void *drafts;  // int32 or int64
  int drafts64;
  int64_t draft_stride;
  const int32_t *parents;
  int64_t parent_stride;  // 0: one tree for all
  const int32_t *counts;  // nullable: nodes
  const int64_t *targets;
  int64_t target_stride;
  const int32_t *seq_lens;  // nullable
  int batch, nodes, width;
  int32_t *path;
  int64_t path_stride;
  int64_t *out_tokens;
  int64_t out_stride;
  int32_t *accepted;
  int32_t *next_lens;  // nullable
};

// x of lane `src`, the same lane for the whole wave.
__device__ __forceinline__ int64_t lane_i64(int64_t x, int src) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(x), src);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(x >> 32), src);
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

__global__ __launch_bounds__(64 * kSeqs) void accept_tree_kernel(AcceptArgs a) {
  const int lane = threadIdx.x & (kWave - 1);
  const int b = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x) * kSeqs + static_cast<int>(threadIdx.x) / kWave);
  if (b >= a.batch) return;
  const int n = min(max(a.counts ? a.counts[b] : a.nodes, 0), a.nodes);
  int64_t draft = -1, target = -1;
  int parent = -1;
  if (lane < n) {
    const int64_t at = b * a.draft_stride + lane;
    draft = a.drafts64 ? static_cast<const int64_t *>(a.drafts)[at] : static_cast<const int32_t *>(a.drafts)[at];
    target = a.targets[b * a.target_stride + lane];
    parent = a.parents[b * a.parent_stride + lane];
  }
  int passed = 0;  // nodes of the walk, the root included
  int mine = -1;   // lane i: the walk's i-th node and the token chosen there
  int64_t token = -1;
  for (int node = 0; n > 0;) {
    const int64_t t = lane_i64(target, node);
    if (lane == passed) {
      mine = node;
      token = t;
    }
    if (++passed == a.width) break;
    // A child lies behind its parent, so the walk ends.
    const uint64_t fits = __ballot(lane > node && parent == node && draft == t && t >= 0);
    if (!fits) break;
    node = __builtin_ctzll(fits);
  }
  if (lane < a.width) {
    a.path[b * a.path_stride + lane] = mine;
    a.out_tokens[b * a.out_stride + lane] = token;
  }
  if (lane == 0) {
    a.accepted[b] = passed - 1;
    if (a.next_lens) a.next_lens[b] = a.seq_lens[b] + passed;
  }
}

}  // namespace
}  // namespace k8v4

extern "C" int k8v4_accept_tree(const void *draft_tokens, int drafts_are_int64, int64_t draft_stride,
                                const int32_t *parents, int64_t parent_stride, const int32_t *num_nodes,
                                const int64_t *target_tokens, int64_t target_stride, const int32_t *seq_lens,
                                int64_t batch, int nodes, int width, int32_t *path, int64_t path_stride,
                                int64_t *out_tokens, int64_t out_stride, int32_t *accepted, int32_t *next_lens,
                                void *stream) {
  using namespace k8v4;
  clear_error();
  K8V4_REQUIRE(nodes >= 1 && nodes <= kMaxNodes, "1 to %d nodes a tree, got %d", kMaxNodes, nodes);
  K8V4_REQUIRE(width >= 1 && width <= nodes, "path width must be 1 .. nodes, got %d", width);
  K8V4_REQUIRE(batch >= 0 && batch < (int64_t(1) << 24), "bad batch");
  if (batch == 0) return K8V4_OK;
  K8V4_REQUIRE(draft_tokens && parents && target_tokens && path && out_tokens && accepted, "null pointer");
  K8V4_REQUIRE(!next_lens || seq_lens, "next_lens needs seq_lens");
  K8V4_REQUIRE(draft_stride >= nodes || batch == 1, "draft_tokens row stride shorter than the nodes");
  K8V4_REQUIRE(parent_stride >= nodes || parent_stride == 0 || batch == 1, "parents row stride shorter than the nodes");
  K8V4_REQUIRE(target_stride >= nodes || batch == 1, "target_tokens row stride shorter than the nodes");
  K8V4_REQUIRE(path_stride >= width || batch == 1, "path row stride shorter than its width");
  K8V4_REQUIRE(out_stride >= width || batch == 1, "out_tokens row stride shorter than its width");
  const auto misaligned = [](const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
  K8V4_REQUIRE(!misaligned(draft_tokens, drafts_are_int64 ? 8 : 4) && !misaligned(parents, 4) &&
                   !misaligned(num_nodes, 4) && !misaligned(target_tokens, 8) && !misaligned(seq_lens, 4) &&
                   !misaligned(path, 4) && !misaligned(out_tokens, 8) && !misaligned(accepted, 4) &&
                   !misaligned(next_lens, 4),
               "misaligned pointer");
  AcceptArgs a;
  a.drafts = draft_tokens;
  a.drafts64 = drafts_are_int64 != 0;
  a.draft_stride = draft_stride;
  a.parents = parents;
  a.parent_stride = parent_stride;
  a.counts = num_nodes;
  a.targets = target_tokens;
  a.target_stride = target_stride;
  a.seq_lens = seq_lens;
  a.batch = static_cast<int>(batch);
  a.nodes = nodes;
  a.width = width;
  a.path = path;
  a.path_stride = path_stride;
  a.out_tokens = out_tokens;
  a.out_stride = out_stride;
  a.accepted = accepted;
  a.next_lens = next_lens;
  accept_tree_kernel<<<dim3(static_cast<unsigned>((batch + kSeqs - 1) / kSeqs)), dim3(64 * kSeqs), 0,
                       static_cast<hipStream_t>(stream)>>>(a);
  return launch_status("k8v4_accept_tree");
}
