// Device code shared by the decode kernels: the LDS image of a chunk of cached
// tokens, the loads that fill it, the score, softmax and output steps over it,
// and the ring's layout.  One query tile is 16 rows; a chunk is 32 tokens of
// one KV head.  The arguments' type A only has to carry the cache description
// (k_cache .. vz_ps, planes_fast, d_kv, d_vz) and, for physical_page, ppb.
#pragma once

#include "k8v4_common.h"

#include <cfloat>

namespace k8v4 {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kScoreBias = 0x4B400000;  // bits of 1.5 * 2^23
// Lazy-rescale threshold (log2 units): the running max m moves only when a
// score passes it by more than 4, so exp2(score - m) <= 16.  P is carried as
// exp2(score - m - 2), a quarter of the probability (row sums and outputs
// shrink alike, so their ratio is unchanged), and is multiplied by the
// token's V scale in fp16: a V row spanning the whole fp16 range has scale
// 2 * 65504 / 15, and 16 / 4 * 2 * 65504 / 15 = 34,936 stays finite.
constexpr float kRescaleThreshold = 4.0f;
constexpr float kPLog2Offset = 2.0f;

// Block-table reads go through the constant address space: the table is
// read-only for the kernel's lifetime, so a uniform lookup becomes a scalar
// load and never waits on the vector-memory counter the LDS DMA uses.
typedef const __attribute__((address_space(4))) int32_t *const_i32_ptr;

template <typename A>
__device__ __forceinline__ int physical_page(const A &a, const int32_t *bt_row, int p) {
  const const_i32_ptr row = (const_i32_ptr)(bt_row);
  if (a.ppb <= 1) return row[p];
  return row[p / a.ppb] * a.ppb + (p % a.ppb);
}

__device__ __forceinline__ void store_out(void *out, int dtype, int64_t idx, float v) {
  if (dtype == K8V4_F32)
    static_cast<float *>(out)[idx] = v;
  else if (dtype == K8V4_BF16)
    static_cast<__bf16 *>(out)[idx] = static_cast<__bf16>(v);
  else
    static_cast<_Float16 *>(out)[idx] = static_cast<_Float16>(v);
}

typedef float v8f __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

typedef __attribute__((address_space(3))) char lds_t;

template <int D>
struct Slot {
  static constexpr int KS = D / 64;     // 64-dim k-steps of the QK MFMA
  static constexpr int DG = D / 128;    // 8-dim dword groups per lane in a V row
  static constexpr int VROW = D / 2;    // bytes of one token's V row (one head)
  static constexpr int KRP = 1024 / D;  // K rows per 1 KB DMA
  // K slot: [32 tokens][D] codes, 16-byte chunks XOR-swizzled per row.
  static constexpr int K_BYTES = 32 * D;
  // V slot: [32 tokens][VROW] V rows (rotated order), then ks[32] | vs[32] | vz[32].
  static constexpr int S_OFF = 32 * VROW;
  static constexpr int V_BYTES = S_OFF + 384;
  static constexpr int NK = 32 * D / 1024;       // 16-byte DMAs for the K rows
  static constexpr int NV = 32 * VROW / 1024;    // 16-byte DMAs for the V rows
  static constexpr int NVS = NV + 2;             // V rows + the two scale-plane DMAs
};

// K rows sit in LDS with their 16-byte chunks permuted: chunk c of row t is at
// position c ^ kswz(t).  A DMA writes lane L at byte 16*L of its 1 KB, so the
// permutation is applied on the source side; it makes the 16 rows read by one
// quarter-wave of the A-operand ds_read_b128 land in 16 distinct bank groups.
// LDS row position of the V row of chunk_token(g, i) (see lane_offsets).
template <int D>
__device__ __forceinline__ int vrow_pos(int g, int i) {
  const int half = i >> 2, ii = i & 3;
  if constexpr (D == 128) return 16 * half + 4 * g + ((ii + g) & 3);
  return 16 * half + 4 * g + ii;
}

template <int D>
__device__ __forceinline__ int kswz(int t) {
  if constexpr (D == 128) return (t & 7) ^ ((t >> 3) & 1);
  return t & 15;
}

// Token (0..31 within the chunk) held in slot i of a lane of group g: the two
// 16-token halves of the transposed QK^T output tile.
__device__ __forceinline__ int chunk_token(int g, int i) { return i < 4 ? 4 * g + i : 16 + 4 * g + (i - 4); }

// Direct-to-LDS loads.  K rows (one 128-byte line per token and head) are
// read exactly once and carry the nontemporal policy (streaming reads
// measured faster on MI355X).  A V row is half of a 128-byte line whose other
// half is the neighbouring head's row, read by another wave of the same
// work-group moments later: with the nontemporal policy that line was often
// fetched twice (HBM reads 1.08x the algorithmic bytes), with the default
// policy once (1.005x) at the same speed.  The scale planes, shared by the
// heads of a work-group, and the query rows, shared by the splits of a
// sequence, also use the default policy.
//
// The loads use the scalar-base form: a wave-uniform 64-bit base in SGPRs
// plus a 32-bit per-lane offset, so issuing one costs no vector instruction
// (the compiler's builtin forms every lane's 64-bit address with vector
// adds).  Written as inline assembly, these loads are invisible to the
// compiler's wait counting: every wait on them is explicit (wait_vm), and a
// compiler-generated wait can only be stronger than needed, never weaker
// (vector loads complete in issue order); nor does the compiler see LDS
// being written, which keeps it from waiting for every load in flight before
// each LDS read.  The compiler's hazard checks do not look inside inline
// assembly, so the statement sets M0 (the LDS destination) itself and then
// waits the states the load needs after a scalar write of M0 (1) and after a
// vector write of an SGPR it reads, such as a v_readfirstlane result in its
// base (5).
__device__ __forceinline__ uint32_t lds_addr(const lds_t *p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p));
}
__device__ __forceinline__ void dma16s_nt(const void *sbase, uint32_t voff, const lds_t *dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(voff), "s"(sbase),
               "s"(lds_addr(dst))
               : "memory", "m0");
}
__device__ __forceinline__ void dma16s(const void *sbase, uint32_t voff, const lds_t *dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase),
               "s"(lds_addr(dst))
               : "memory", "m0");
}
// Per-lane 64-bit addresses (no scalar base): same statement shape.
__device__ __forceinline__ void dma4v(const void *addr, const lds_t *dst) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 4\n\tglobal_load_lds_dword %0, off" ::"v"(addr), "s"(lds_addr(dst))
               : "memory", "m0");
}
__device__ __forceinline__ void dma4s(const void *sbase, uint32_t voff, const lds_t *dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dword %0, %1" ::"v"(voff), "s"(sbase),
               "s"(lds_addr(dst))
               : "memory", "m0");
}

// Split-state stores at device scope (sc1): written through the XCD's L2 to
// memory, where the merge kernel reads them.  With default stores the states
// of the work-groups that finish last are still dirty in L2 when the kernel
// ends, and the end-of-kernel write-back of them delays the merge launch
// (4 x 8,192 tokens, q = 7: 1.5 us per step).  Vector stores; they are the
// last memory operations of the kernel, so the compiler's wait counting, which
// does not see them, has nothing after them to order.  Its hazard checks do
// not see them either: a store of more than 8 bytes still reads its data
// registers after issue, so the statement itself waits the states before a
// later instruction may overwrite them (s_nop 1).
__device__ __forceinline__ void store_wt16(void *dst, v8h v) {
  asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" ::"v"(dst), "v"(v) : "memory");
}
__device__ __forceinline__ void store_wt8(float2 *dst, float2 v) {
  typedef float v2f_t __attribute__((ext_vector_type(2)));
  const v2f_t x = {v.x, v.y};
  asm volatile("global_store_dwordx2 %0, %1, off sc1\n\ts_nop 1" ::"v"(dst), "v"(x) : "memory");
}

// Per-lane byte offsets of one chunk's DMA sources (loop-invariant).
struct LaneOffsets {
  uint32_t k[4];  // K source per DMA index mod 4: row L/(D/16) of the piece, swizzled chunk
  uint32_t v;     // V: token (lane*16)/VROW (+rows of later DMAs), 16-byte column
  uint32_t s;     // scale plane cell of token (lane & 31)
  // Scalar-base form of the two scale-plane gathers (when the three planes
  // share one page stride): offsets from the lower of the two plane bases a
  // gather reads, lanes 0-31 in the first plane, lanes 32-63 in the second.
  uint32_t sa, sb;
};

// PH (paired halves, head dim 256 served as two 128-dim halves): h and HKV
// count half-heads; the scale planes belong to the whole head h / 2 of HKV / 2.
template <int D, int HKV, bool PH = false, typename A>
__device__ __forceinline__ LaneOffsets lane_offsets(const A &a, int h, int lane) {
  constexpr int VROW = D / 2, KRP = 1024 / D, CPR = D / 16;
  constexpr int HS = PH ? HKV / 2 : HKV;  // heads of the scale planes
  LaneOffsets o;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int t = j * KRP + lane / CPR;  // row of DMA j (mod 4) this lane fills
    const int c = (lane % CPR) ^ kswz<D>(t);
    o.k[j] = static_cast<uint32_t>((lane / CPR) * (HKV * D) + h * D + 16 * c);
  }
  {
    // V rows of one DMA sit in LDS rotated within groups of four rows
    // (position 4q + ((i + q) & 3) holds row 4q + i) so the eight 4-byte
    // operand reads of a chunk spread over all banks.
    const int pos = (lane * 16) / VROW;
    const int row = VROW == 64 ? 4 * (pos >> 2) + (((pos & 3) - (pos >> 2)) & 3) : pos;
    o.v = static_cast<uint32_t>(row * (HKV * VROW) + h * VROW + (lane * 16) % VROW);
  }
  o.s = static_cast<uint32_t>(((lane & 31) * HS + (PH ? h >> 1 : h)) * 4);
  const int64_t lo_kv = a.d_kv < 0 ? a.d_kv : 0, lo_vz = a.d_vz < 0 ? a.d_vz : 0;
  o.sa = o.s + static_cast<uint32_t>(lane < 32 ? -lo_kv : a.d_kv - lo_kv);
  o.sb = o.s + static_cast<uint32_t>(lane < 32 ? -lo_vz : a.d_vz - lo_vz);
  return o;
}

// Starts the DMA of chunk x (32 tokens of head h, in physical page `phys`, -1
// outside the cache) into `slot`; returns whether the page is a cache page.
// An invalid page still issues its loads (from page 0) so every chunk costs
// the same vmcnt.  K and V move in
// 16-byte-per-lane DMAs from a wave-uniform base plus a 32-bit lane offset;
// the scale planes of this head are gathered with two 4-byte DMAs (lanes
// 0-31: k_scale then v_scale, lanes 32-63: v_scale then v_zero).
template <int D, int HKV, typename A>
__device__ __forceinline__ int issue_k(const A &a, int phys, int x, const LaneOffsets &lo, lds_t *kslot) {
  using S = Slot<D>;
  const int half = x & 1;
  const int valid = phys >= 0 ? 1 : 0;
  if (!valid) phys = 0;
  const char *kb = reinterpret_cast<const char *>(a.k_cache) + phys * a.k_ps +
                   static_cast<int64_t>(32 * half) * HKV * D;
#pragma unroll
  for (int j = 0; j < S::NK; ++j) dma16s_nt(kb + static_cast<int64_t>(j) * S::KRP * (HKV * D), lo.k[j & 3], kslot + j * 1024);
  return valid;
}

template <int D, int HKV, bool PH = false, typename A>
__device__ __forceinline__ void issue_v(const A &a, int phys, int x, const LaneOffsets &lo, int lane,
                                        lds_t *vslot) {
  using S = Slot<D>;
  constexpr int HS = PH ? HKV / 2 : HKV;  // heads of the scale planes
  const int half = x & 1;
  if (phys < 0) phys = 0;
  const int tok0 = 32 * half;
  const char *vb = reinterpret_cast<const char *>(a.v_cache) + phys * a.v_ps +
                   static_cast<int64_t>(tok0) * HKV * S::VROW;
#pragma unroll
  for (int j = 0; j < S::NV; ++j) dma16s(vb + static_cast<int64_t>(j) * (1024 / S::VROW) * (HKV * S::VROW), lo.v, vslot + j * 1024);
  // Two full-wave 4-byte DMAs, no divergent branch: ks[32] | vs[32] at
  // S_OFF, then vs[32] | vz[32] at S_OFF + 128 (the v_scale cells are written
  // twice with the same values).
  const int64_t plane0 = static_cast<int64_t>(tok0) * HS * 4;
  if (a.planes_fast) {
    const int64_t lo_kv = a.d_kv < 0 ? a.d_kv : 0, lo_vz = a.d_vz < 0 ? a.d_vz : 0;
    const char *pa = reinterpret_cast<const char *>(a.k_scale) + lo_kv + phys * a.ks_ps + plane0;
    const char *pb = reinterpret_cast<const char *>(a.v_scale) + lo_vz + phys * a.vs_ps + plane0;
    dma4s(pa, lo.sa, vslot + S::S_OFF);
    dma4s(pb, lo.sb, vslot + S::S_OFF + 128);
  } else {
    const char *ksp = reinterpret_cast<const char *>(a.k_scale) + phys * a.ks_ps + plane0 + lo.s;
    const char *vsp = reinterpret_cast<const char *>(a.v_scale) + phys * a.vs_ps + plane0 + lo.s;
    const char *vzp = reinterpret_cast<const char *>(a.v_zero) + phys * a.vz_ps + plane0 + lo.s;
    dma4v(lane < 32 ? ksp : vsp, vslot + S::S_OFF);
    dma4v(lane < 32 ? vsp : vzp, vslot + S::S_OFF + 128);
  }
}

// Wait until at most `after` chunks' DMAs are still in flight.
// Wait until at most n (wave-uniform, 0..) vector-memory loads are
// outstanding.  s_waitcnt takes an immediate, so the count is dispatched;
// counts above 62 wait for 62 (more than needed, still correct).
__device__ __forceinline__ void wait_vm(int n) {
#define K8V4_WAIT_CASE(N) \
  case N:                 \
    asm volatile("s_waitcnt vmcnt(" #N ")" ::: "memory"); \
    break;
  switch (n < 62 ? n : 62) {
    K8V4_WAIT_CASE(0) K8V4_WAIT_CASE(1) K8V4_WAIT_CASE(2) K8V4_WAIT_CASE(3) K8V4_WAIT_CASE(4)
    K8V4_WAIT_CASE(5) K8V4_WAIT_CASE(6) K8V4_WAIT_CASE(7) K8V4_WAIT_CASE(8) K8V4_WAIT_CASE(9)
    K8V4_WAIT_CASE(10) K8V4_WAIT_CASE(11) K8V4_WAIT_CASE(12) K8V4_WAIT_CASE(13) K8V4_WAIT_CASE(14)
    K8V4_WAIT_CASE(15) K8V4_WAIT_CASE(16) K8V4_WAIT_CASE(17) K8V4_WAIT_CASE(18) K8V4_WAIT_CASE(19)
    K8V4_WAIT_CASE(20) K8V4_WAIT_CASE(21) K8V4_WAIT_CASE(22) K8V4_WAIT_CASE(23) K8V4_WAIT_CASE(24)
    K8V4_WAIT_CASE(25) K8V4_WAIT_CASE(26) K8V4_WAIT_CASE(27) K8V4_WAIT_CASE(28) K8V4_WAIT_CASE(29)
    K8V4_WAIT_CASE(30) K8V4_WAIT_CASE(31) K8V4_WAIT_CASE(32) K8V4_WAIT_CASE(33) K8V4_WAIT_CASE(34)
    K8V4_WAIT_CASE(35) K8V4_WAIT_CASE(36) K8V4_WAIT_CASE(37) K8V4_WAIT_CASE(38) K8V4_WAIT_CASE(39)
    K8V4_WAIT_CASE(40) K8V4_WAIT_CASE(41) K8V4_WAIT_CASE(42) K8V4_WAIT_CASE(43) K8V4_WAIT_CASE(44)
    K8V4_WAIT_CASE(45) K8V4_WAIT_CASE(46) K8V4_WAIT_CASE(47) K8V4_WAIT_CASE(48) K8V4_WAIT_CASE(49)
    K8V4_WAIT_CASE(50) K8V4_WAIT_CASE(51) K8V4_WAIT_CASE(52) K8V4_WAIT_CASE(53) K8V4_WAIT_CASE(54)
    K8V4_WAIT_CASE(55) K8V4_WAIT_CASE(56) K8V4_WAIT_CASE(57) K8V4_WAIT_CASE(58) K8V4_WAIT_CASE(59)
    K8V4_WAIT_CASE(60) K8V4_WAIT_CASE(61)
    default:
      asm volatile("s_waitcnt vmcnt(62)" ::: "memory");
      break;
  }
#undef K8V4_WAIT_CASE
}

__device__ __forceinline__ v2h pack_h2(float lo, float hi) {
  return __builtin_convertvector((v2f){lo, hi}, v2h);
}

// max(x, x from lane^16) and max(x, x from lane^32) without LDS.
__device__ __forceinline__ float xlane_max16_32(float x) {
  auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r16[0]), __uint_as_float(r16[1]));
  auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r32[0]), __uint_as_float(r32[1]));
}

// (The int8 query operands live in LDS, shared by the waves of a head.)
template <int D, int NT>
struct WaveState {
  static constexpr int DG = D / 128;
  float crow[NT];   // q_scale * log2(e) / sqrt(D), > 0
  int lim[NT];      // causal end of this lane's row (S layout)
  float m_run[NT];  // running max, log2 domain (S layout)
  float thr[NT];    // (m_run + threshold) / crow: a raw score above it moves m_run
  v4f lsum[NT];     // row sums (O layout, rows 4g+i)
  v4f corr[NT];     // sum of P * v_scale * v_zero per row (O layout)
  v4f O[NT][DG][8]; // unnormalized output (O layout)
};

// TS: LDS tiles between this wave's query tiles (2 when the waves of a head
// hold alternate row tiles).
template <int D, int NT, int TS = 1>
__device__ __forceinline__ void chunk_qk(const lds_t *kslot, const lds_t *qlds, int lane, int g, v4i (&sc)[2][NT]) {
  using S = Slot<D>;
  constexpr int KS = S::KS;
  // ---- QK^T, transposed: S[ml][nt] lane (n,g) reg i = score(token 16*ml+4g+i, row 16*nt+n)
  v4i kf[2][KS];
  const int n = lane & 15;
#pragma unroll
  for (int ml = 0; ml < 2; ++ml)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int t = 16 * ml + n, c = 4 * ks + g;
      kf[ml][ks] = *reinterpret_cast<const __attribute__((address_space(3))) v4i *>(
          kslot + t * D + 16 * (c ^ kswz<D>(t)));
    }
  // k-step outermost: the 2 * NT score tiles are independent accumulators,
  // so consecutive MFMAs never wait on each other.
#pragma unroll
  for (int ml = 0; ml < 2; ++ml)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sc[ml][nt] = (v4i){kScoreBias, kScoreBias, kScoreBias, kScoreBias};
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const v4i qf =
          *reinterpret_cast<const __attribute__((address_space(3))) v4i *>(qlds + ((nt * TS * KS + ks) * kWave + lane) * 16);
#pragma unroll
      for (int ml = 0; ml < 2; ++ml) sc[ml][nt] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[ml][ks], qf, sc[ml][nt], 0, 0, 0);
    }
}

// QK^T of a 256-dim head from two 128-dim K slots (paired halves): dims
// 0-127 of the chunk's keys in `klo`, dims 128-255 in `khi` (the slots of the
// two waves of the pair), the query fragments of all four 64-dim k-steps in
// LDS.  Same score layout and bias as chunk_qk; |dot| <= 256 * 127 * 127 <
// 2^22 keeps the biased accumulator exact.  The two halves' K operands are
// read one half at a time (16 registers instead of 32).
template <int NT, int TS = 1>
__device__ __forceinline__ void chunk_qk_pair(const lds_t *klo, const lds_t *khi, const lds_t *qlds, int lane, int g,
                                              v4i (&sc)[2][NT]) {
  const int n = lane & 15;
#pragma unroll
  for (int ml = 0; ml < 2; ++ml)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sc[ml][nt] = (v4i){kScoreBias, kScoreBias, kScoreBias, kScoreBias};
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const lds_t *kslot = part ? khi : klo;
    v4i kf[2][2];
#pragma unroll
    for (int ml = 0; ml < 2; ++ml)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const int t = 16 * ml + n, c = 4 * ks + g;
        kf[ml][ks] = *reinterpret_cast<const __attribute__((address_space(3))) v4i *>(
            kslot + t * 128 + 16 * (c ^ kswz<128>(t)));
      }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const v4i qf = *reinterpret_cast<const __attribute__((address_space(3))) v4i *>(
            qlds + ((nt * TS * 4 + 2 * part + ks) * kWave + lane) * 16);
#pragma unroll
        for (int ml = 0; ml < 2; ++ml) sc[ml][nt] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[ml][ks], qf, sc[ml][nt], 0, 0, 0);
      }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Flags of the paired-halves handshake, one word per wave in LDS.  A flag
// only grows within a launch; a wait polls its partner's word (wave-uniform)
// until it reaches the target, sleeping between polls.  The pair runs the
// same chunk sequence and neither wave waits before publishing what the
// other waits for, so every wait ends; the bound only caps a wait that a
// broken launch could otherwise make endless, and such a give-up is counted
// in a device word the host reads (k8v4_decode_fault_count), so it shows up
// in tests instead of as a silently wrong output.
typedef __attribute__((address_space(3))) int lds_int;
__device__ int g_pair_wait_timeouts;
__device__ __forceinline__ void pair_flag_set(lds_int *f, int v, int lane) {
  if (lane == 0) *reinterpret_cast<volatile lds_int *>(f) = v;
}
__device__ __forceinline__ void pair_flag_wait(const lds_int *f, int target, int lane) {
  for (int it = 0; it < (1 << 22); ++it) {
    const int v = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const volatile lds_int *>(f));
    if (v >= target) return;
    __builtin_amdgcn_s_sleep(1);
  }
  if (lane == 0) __hip_atomic_fetch_add(&g_pair_wait_timeouts, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// What rows of a drafted tree see: the tokens ahead of `context`, and of the tree's
// tokens behind them those whose bit is set in the row's word (row r's is words[r / 6]).
// A token of the tree that none of the `count` words has may never have been stored:
// its planes may hold anything and are not used.
struct TreeRows {
  const __attribute__((address_space(3))) uint64_t *words;
  int context, count;
};

// Softmax and P.V of one chunk whose scores chunk_qk produced; reads the V
// rows and scale planes of the chunk's V slot.  A row sees the tokens ahead of
// its st.lim, or (TREE) what `tree` says.
template <int D, int NT, bool RAISE = false, bool TREE = false>
__device__ __forceinline__ void chunk_softmax_pv(WaveState<D, NT> &st, const v4i (&sc)[2][NT],
                                                 const lds_t *vslot, int tbase, int L0, int lane, int g,
                                                 bool masked, TreeRows tree = {}) {
  using S = Slot<D>;
  constexpr int DG = S::DG;
  // Phase fences keep the scheduler from hoisting later LDS reads into this
  // phase, which would raise register pressure past two waves per SIMD.
  __builtin_amdgcn_sched_barrier(0);
  // RAISE (the paired halves): the softmax's vector work runs at a raised
  // issue priority, so beside the other wave's matrix phases it overlaps them
  // instead of queueing behind that wave's vector instructions (reference
  // shape 40.6 -> 40.2 us; with the 128-dim kernels' progress balance it
  // measured slower at the headline, so they do not raise).
  if constexpr (RAISE) __builtin_amdgcn_s_setprio(1);
  // ---- scale planes of this lane's 8 tokens: [0..3] = tokens 4g+i, [4..7] = 16+4g+i
  typedef float v4f_l __attribute__((ext_vector_type(4)));
  const auto *sp = reinterpret_cast<const __attribute__((address_space(3))) v4f_l *>(vslot + S::S_OFF);
  v4f_l ksa = sp[g], ksb = sp[4 + g], vsa = sp[8 + g], vsb = sp[12 + g], vza = sp[16 + g], vzb = sp[20 + g];
  float ksv[8] = {ksa[0], ksa[1], ksa[2], ksa[3], ksb[0], ksb[1], ksb[2], ksb[3]};
  float vsv[8] = {vsa[0], vsa[1], vsa[2], vsa[3], vsb[0], vsb[1], vsb[2], vsb[3]};
  float vzv[8] = {vza[0], vza[1], vza[2], vza[3], vzb[0], vzb[1], vzb[2], vzb[3]};
  if (__builtin_expect(masked, 0)) {
    [[maybe_unused]] uint64_t any = 0;  // nodes that some row sees
    if constexpr (TREE) {
      for (int i = 0; i < tree.count; ++i) any |= tree.words[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bool unused = tbase + chunk_token(g, i) >= L0;  // unwritten tail: never use its planes
      if constexpr (TREE) {
        const int node = tbase + chunk_token(g, i) - tree.context;
        unused |= node >= 0 && !((any >> (node & 63)) & 1);
      }
      if (unused) {
        ksv[i] = 0.f;
        vsv[i] = 0.f;
        vzv[i] = 0.f;
      }
    }
  }
  // The QK accumulators start at the bits of 1.5 * 2^23, so each reads as the
  // float 12582912 + dot, exactly (|dot| <= 128 * 127 * 127 < 2^22); one fma
  // with k_bias = -12582912 * k_scale gives dot * k_scale within 0.75 of a
  // unit of the dot (the rounding of k_bias) -- against a query quantization
  // step of about 0.3 * |k| per dim.
  float kbias[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) kbias[i] = -12582912.0f * ksv[i];
  // ---- scores, chunk max, lazy rescale
  float t[2][NT][4];
  float lmx[NT];  // this lane's largest score of each row tile
  bool grow = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float mx = -INFINITY;
#pragma unroll
    for (int ml = 0; ml < 2; ++ml)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v = fmaf(__int_as_float(sc[ml][nt][i]), ksv[4 * ml + i], kbias[4 * ml + i]);
        t[ml][nt][i] = v;
      }
    if (__builtin_expect(masked, 0)) {
      if constexpr (TREE) {
        const uint64_t word = tree.words[(16 * nt + (lane & 15)) / kGqa];
#pragma unroll
        for (int ml = 0; ml < 2; ++ml)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int tok = tbase + 16 * ml + 4 * g + i, node = tok - tree.context;
            if (tok >= L0 || (node >= 0 && !((word >> (node & 63)) & 1))) t[ml][nt][i] = -INFINITY;
          }
      } else {
#pragma unroll
        for (int ml = 0; ml < 2; ++ml)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (tbase + 16 * ml + 4 * g + i >= st.lim[nt]) t[ml][nt][i] = -INFINITY;
      }
    }
#pragma unroll
    for (int ml = 0; ml < 2; ++ml)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, t[ml][nt][i]);
    lmx[nt] = mx;
    // A row's largest score passes the threshold exactly when one of its four
    // lanes' does, so the cross-lane max is only taken on a rescale.
    grow |= mx > st.thr[nt];
  }
  if (__ballot(grow)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float mnew = fmaxf(st.m_run[nt], xlane_max16_32(lmx[nt]) * st.crow[nt]);
      const float alpha = st.m_run[nt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m_run[nt] - mnew);
      st.m_run[nt] = mnew;
      st.thr[nt] = (mnew + kRescaleThreshold) / st.crow[nt];
      float ai[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ai[i] = __shfl(alpha, 4 * g + i, kWave);
        st.lsum[nt][i] *= ai[i];
        st.corr[nt][i] *= ai[i];
      }
#pragma unroll
      for (int dg = 0; dg < DG; ++dg)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) st.O[nt][dg][j][i] *= ai[i];
    }
  }
  // ---- P = exp2(score * c - m), packed fp16 in the PV A-operand layout; row sums by MFMA
  const v8h ones = {1, 1, 1, 1, 1, 1, 1, 1};
  v2h vsp[4];
  v8h bz;  // v_zero of the lane's tokens: the zero-point correction operand
  {
    const v2h z01 = pack_h2(vzv[0], vzv[1]), z23 = pack_h2(vzv[2], vzv[3]);
    const v2h z45 = pack_h2(vzv[4], vzv[5]), z67 = pack_h2(vzv[6], vzv[7]);
    bz = (v8h){z01[0], z01[1], z23[0], z23[1], z45[0], z45[1], z67[0], z67[1]};
#pragma unroll
    for (int qp = 0; qp < 4; ++qp) vsp[qp] = pack_h2(vsv[2 * qp], vsv[2 * qp + 1]);
  }
  v8h PA[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float nm = -fmaxf(st.m_run[nt], -FLT_MAX) - kPLog2Offset;
    float p[8];
#pragma unroll
    for (int ml = 0; ml < 2; ++ml)
#pragma unroll
      for (int i = 0; i < 4; ++i) p[4 * ml + i] = __builtin_amdgcn_exp2f(fmaf(t[ml][nt][i], st.crow[nt], nm));
    v2h pp[4] = {pack_h2(p[0], p[1]), pack_h2(p[2], p[3]), pack_h2(p[4], p[5]), pack_h2(p[6], p[7])};
    st.lsum[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
        (v8h){pp[0][0], pp[0][1], pp[1][0], pp[1][1], pp[2][0], pp[2][1], pp[3][0], pp[3][1]}, ones, st.lsum[nt],
        0, 0, 0);
    // P' = P * v_scale of each token (the V scale moves onto the A operand).
#pragma unroll
    for (int qp = 0; qp < 4; ++qp) pp[qp] = pp[qp] * vsp[qp];
    PA[nt] = (v8h){pp[0][0], pp[0][1], pp[1][0], pp[1][1], pp[2][0], pp[2][1], pp[3][0], pp[3][1]};
    st.corr[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(PA[nt], bz, st.corr[nt], 0, 0, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (RAISE) __builtin_amdgcn_s_setprio(0);
  // ---- V: the packed bytes themselves are the B operand, read as fp16
  // subnormals: a byte in the low half of a 16-bit lane is (16 hi + lo) * 2^-24
  // and (x & 0x00F000F0) is hi * 2^-20.  Exact; the finalization takes the
  // even dim as the difference, rescales by 2^24 / 2^20 and subtracts the
  // zero-point correction.
#pragma unroll
  for (int dg = 0; dg < DG; ++dg) {
    uint32_t vw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      vw[i] = *reinterpret_cast<const __attribute__((address_space(3))) uint32_t *>(
          vslot + vrow_pos<D>(g, i) * S::VROW + 64 * dg + 4 * (lane & 15));
#pragma unroll
    for (int byte = 0; byte < 4; ++byte) {
      const uint32_t sel = 0x0C000C00u | (static_cast<uint32_t>(4 + byte) << 16) | static_cast<uint32_t>(byte);
      uint32_t be[4], bo[4];
#pragma unroll
      for (int qp = 0; qp < 4; ++qp) {
        const uint32_t xw = __builtin_amdgcn_perm(vw[2 * qp + 1], vw[2 * qp], sel);
        be[qp] = xw;
        bo[qp] = xw & 0x00F000F0u;
      }
      const v8h Be = __builtin_bit_cast(v8h, (v4i){static_cast<int>(be[0]), static_cast<int>(be[1]),
                                                   static_cast<int>(be[2]), static_cast<int>(be[3])});
      const v8h Bo = __builtin_bit_cast(v8h, (v4i){static_cast<int>(bo[0]), static_cast<int>(bo[1]),
                                                   static_cast<int>(bo[2]), static_cast<int>(bo[3])});
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        st.O[nt][dg][2 * byte] = __builtin_amdgcn_mfma_f32_16x16x32_f16(PA[nt], Be, st.O[nt][dg][2 * byte], 0, 0, 0);
        st.O[nt][dg][2 * byte + 1] =
            __builtin_amdgcn_mfma_f32_16x16x32_f16(PA[nt], Bo, st.O[nt][dg][2 * byte + 1], 0, 0, 0);
      }
    }
  }
}

// O = sum P' * q * 2^-24 (even dims) or 2^-20 (odd dims); the dequantized
// value is (q - zero) * scale, so the true accumulator is the rescaled sum
// minus the zero-point correction.
template <int D, int NT>
__device__ __forceinline__ void finalize_output(WaveState<D, NT> &st) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int dg = 0; dg < D / 128; ++dg)
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        // O[j] holds sum p' (16 hi + lo) 2^-24 (the whole byte), O[j+1] holds
        // sum p' 16 hi 2^-24: the even dim is their difference.
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float whole = st.O[nt][dg][j][i], high = st.O[nt][dg][j + 1][i];
          st.O[nt][dg][j][i] = fmaf(whole - high, 16777216.0f, -st.corr[nt][i]);
          st.O[nt][dg][j + 1][i] = fmaf(high, 1048576.0f, -st.corr[nt][i]);
        }
      }
}

template <int D, int NT, int HKV, int NWH, bool PH = false, bool RS = false>
struct SplitConfig {
  // Two waves per head (NWH = 2), or paired halves (PH) with one or two
  // waves per half-head; two waves per SIMD either way.  The int8 Q operands
  // live in LDS, per head (shared by its waves; PH: all 256 dims, per whole
  // head).  Each wave owns a K ring of RK slots and a V ring of RV slots,
  // the K ring as deep as the LDS allows; a K slot is refilled as soon as
  // its QK^T product is issued, so while a wave computes one chunk up to
  // RK - 1 K slots and RV - 1 V slots are in flight.  PH: D = 128 and HKV
  // half-heads serve a 256-dim cache of HKV / 2 heads.  RS (row split, four
  // row tiles): the two waves of a head hold alternate row tiles (NT each)
  // and both multiply every chunk of the split, each chunk resident in the
  // ring of the wave that loaded it.
  static constexpr int NTQ = RS ? 2 * NT : NT;    // row tiles of a head's query
  static constexpr int DQ = PH ? 2 * D : D;       // dims of one score
  static constexpr int QHEADS = PH ? HKV / 2 : HKV;
  static constexpr int WAVES = HKV * NWH;
  static constexpr int Q_FRAG_BYTES = NTQ * (DQ / 64) * kWave * 16;       // int8 B-operand fragments
  static constexpr int Q_LDS_BYTES = Q_FRAG_BYTES + NTQ * 16 * 4;          // + per-row factors
  // 4 / HKV work-groups share a CU (the grid is about that many per CU; one
  // with eight half-head waves).
  static constexpr int LDS_MAX = HKV >= 4 ? 163840 : 163840 * HKV / 4;
  static constexpr int Q_BYTES_PER_HEAD = Q_LDS_BYTES;
  static constexpr int Q_TOTAL = QHEADS * Q_BYTES_PER_HEAD;
  // PH handshake words: per wave, the chunks whose K half is resident and
  // the chunks whose K slots it has finished reading.
  // Progress balance (two waves per head, eight waves: waves w and w + 4
  // share a SIMD): one chunk counter per wave.
  static constexpr bool BALANCE = NWH == 2 && WAVES == 8 && !PH && !RS;
  static constexpr int FLAG_BYTES = (PH || RS) ? 2 * WAVES * 4 : (BALANCE ? WAVES * 4 : 0);
  // A PH wave refills its K slot after P.V, next to the V slot: the other
  // half of its pair reads that slot during its own QK^T.
  static constexpr bool K_EARLY = !PH && !RS;
  static constexpr int RV = 2;
  static constexpr int RK_FIT = ((LDS_MAX - Q_TOTAL - FLAG_BYTES) / WAVES - RV * Slot<D>::V_BYTES) / Slot<D>::K_BYTES;
  static constexpr int RK = RK_FIT < 2 ? 2 : (RK_FIT > 4 ? 4 : RK_FIT);
  static constexpr int WAVE_BYTES = RK * Slot<D>::K_BYTES + RV * Slot<D>::V_BYTES;
  // Loads issued after a chunk's V group until that chunk is consumed, in
  // the steady state of the main loop (one K and one V group per chunk).
  static constexpr int STEADY_AFTER = (RV - 1) * (Slot<D>::NK + Slot<D>::NVS);
  static constexpr int Q_OFF = WAVES * WAVE_BYTES;
  static constexpr int FLAG_OFF = Q_OFF + Q_TOTAL;
  static constexpr int RING_BYTES = FLAG_OFF + FLAG_BYTES;
  // Partner-wave state exchange at the end (reuses the ring memory).
  static constexpr int XCHG_FLOATS = (NT * (D / 128) * 8 * 4 + NT * 4 + NT) * kWave;
  static constexpr int XCHG_BYTES = (NWH > 1 && !RS) ? HKV * XCHG_FLOATS * 4 : 0;
  static constexpr int LDS_BYTES = RING_BYTES > XCHG_BYTES ? RING_BYTES : XCHG_BYTES;
  static constexpr int OCC = HKV > 4 ? HKV * NWH / 4 : NWH;  // waves per SIMD the kernel is built for
  static_assert(LDS_BYTES <= LDS_MAX, "decode ring exceeds the LDS");
  static_assert(PH || NWH == 2, "128-dim heads run two waves each");
  static_assert(!RS || NWH == 2, "row split: two waves per (half-)head");
  // The query rows of a wave's tiles are staged in its K slots 1..RK-1 (RS:
  // loaded into registers instead; PH: read already quantized).
  static_assert(PH || RS || ((NT + NWH - 1) / NWH) * 16 * 2 * D <= (RK - 1) * Slot<D>::K_BYTES,
                "query staging does not fit the K ring");
};

// ------------------------------------------------------------ folding states
// A split's state of one query row is (m, l, O / l): running max (log2), sum
// and a quarter of the normalized output.  A merge thread owns eight dims of a
// row and folds the states of several splits online.

constexpr int kMergeMU = 8;  // splits loaded together by one merge thread

// Running (max, sum, output) of one column, folded online.
struct MergeAcc {
  float M, l;
  v8f o;
};

// One round of a merge thread: the (m, l, O) of its splits s = s0 + u * SPI
// (u < kMergeMU) below `limit`, others empty.
struct MergeRound {
  float ms[kMergeMU], ls[kMergeMU];
  v8f os[kMergeMU];
};

__device__ __forceinline__ void merge_fold_round(MergeAcc &acc, const MergeRound &rd) {
  float mn = acc.M;
#pragma unroll
  for (int u = 0; u < kMergeMU; ++u) mn = fmaxf(mn, rd.ms[u]);
  if (mn != -INFINITY) {
    const float c = acc.M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(acc.M - mn);
    acc.l *= c;
    acc.o *= c;
#pragma unroll
    for (int u = 0; u < kMergeMU; ++u) {
      const float w = rd.ms[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(rd.ms[u] - mn) * rd.ls[u];
      acc.l += w;
      acc.o += (4.f * w) * rd.os[u];  // the states hold a quarter of the split's output
    }
    acc.M = mn;
  }
}

// Rescales an accumulator to the reference max Mr (Mr >= M; both -inf: empty).
__device__ __forceinline__ void merge_rescale(MergeAcc &x, float Mr) {
  const float w = x.M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.M - Mr);
  x.l *= w;
  x.o *= w;
  x.M = Mr;
}

}  // namespace
}  // namespace k8v4
