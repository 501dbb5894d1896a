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
// filled by direct-to-LDS loads, see decode_chunk.h and decode.hip.
#include "decode_chunk.h"

#include <type_traits>

namespace k8v4 {
namespace {

constexpr int kGroup = 8;  // tokens of one segment: 48 rows of a KV head
// Fixed cost of a piece in pages of its pages' time.
constexpr int kPieceCost = 6;
constexpr int kFar = 1 << 30;

struct SharedArgs {
  const int8_t *q8;  // quantized query rows [hkv][head_rows][head_dim]
  const float *q8_scale;
  int64_t head_rows;
  const int8_t *k_cache;
  const float *k_scale;
  const uint8_t *v_cache;
  const float *v_scale;
  const float *v_zero;
  int64_t num_pages;
  int64_t k_ps, ks_ps, v_ps, vs_ps, vz_ps;  // page strides, bytes
  int planes_fast;                          // see DecodeArgs in decode.hip
  int64_t d_kv, d_vz;
  const int32_t *prefix_table;
  int prefix_pages;
  const int32_t *block_table;
  int64_t bt_stride;
  int table_pages;  // pages a table row covers
  int ppb;
  const int32_t *seq_lens;
  int batch, q_len, hkv;
  int tokens;      // batch * q_len
  int groups;      // prefix segments (0 without a prefix)
  int wide_blocks; // many-rows kernel: row blocks of a KV head, groups = hkv * wide_blocks (0: not used)
  int per_seq;     // own segments of a sequence: 1, or 2 for more than eight tokens
  int grid;        // work-groups of the split launch
  char *ws, *own_ws;  // states of the prefix's pieces and of the sequences' own
  int prefix_rows, own_rows;        // state rows of a KV head in a piece of either kind
  int64_t prefix_bytes, own_bytes;  // bytes of such a state
  int merge_cs;    // column slices per output row in the merge
  void *out;
  int out_dtype;
  int64_t out_tok_stride;  // elements
};

// Length of sequence b's own segments on the axis: its pages behind the
// prefix and the fixed cost, or nothing.
__device__ __forceinline__ int own_pages(const SharedArgs &a, int len) {
  const int pages = len > 0 ? min(static_cast<int>((static_cast<int64_t>(len) + kPage - 1) / kPage), a.table_pages) : 0;
  return max(pages - a.prefix_pages, 0);
}
__device__ __forceinline__ int own_cost(const SharedArgs &a, int len) {
  const int n = own_pages(a, len);
  return n > 0 ? n + kPieceCost : 0;
}
__device__ __forceinline__ int prefix_cost(const SharedArgs &a) { return a.prefix_pages + kPieceCost; }

// Units of the axis that one work-group takes, and the units ahead of
// sequence `b` among the own segments.
struct Axis {
  int unit;
  int before;
};
__device__ Axis plan_axis(const SharedArgs &a, int lane, int b) {
  int own = 0, before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kWave) {
    const int i = b0 + lane;
    const int c = i < a.batch ? own_cost(a, a.seq_lens[i]) * a.per_seq : 0;
    own += c;
    before += i < b ? c : 0;
  }
  Axis x;
  const int total = a.groups * prefix_cost(a) + wave_sum(own);
  x.unit = __builtin_amdgcn_readfirstlane(max(1, (total + a.grid - 1) / a.grid));
  x.before = wave_sum(before);
  return x;
}

// The segment that holds unit u of the axis (or the first one behind it) and
// where that segment begins; segments 0 .. groups - 1 are the prefix's.
struct Where {
  int seg;
  int base;
};
__device__ Where locate(const SharedArgs &a, int lane, int u) {
  Where w;
  const int pre = a.groups * prefix_cost(a);
  if (u < pre) {
    w.seg = u / prefix_cost(a);
    w.base = w.seg * prefix_cost(a);
    return w;
  }
  int base = pre;
  for (int b0 = 0; b0 < a.batch; b0 += kWave) {
    const int i = b0 + lane;
    const int c = i < a.batch ? own_cost(a, a.seq_lens[i]) : 0;
    const int incl = base + wave_inclusive_scan(c * a.per_seq);
    const uint64_t past = __ballot(i < a.batch && incl > u);
    if (past) {
      const int src = __builtin_ctzll(past);
      const int cost = __builtin_amdgcn_readlane(c, src);
      const int first = __builtin_amdgcn_readlane(incl, src) - cost * a.per_seq;
      const int sub = u >= first + cost ? 1 : 0;  // at most two segments a sequence
      w.seg = __builtin_amdgcn_readfirstlane(a.groups + (b0 + src) * a.per_seq + sub);
      w.base = __builtin_amdgcn_readfirstlane(first + sub * cost);
      return w;
    }
    base = __builtin_amdgcn_readlane(incl, kWave - 1);
  }
  w.seg = a.groups + a.batch * a.per_seq;
  w.base = base;
  return w;
}

// State of the piece that work-group g makes of a segment.  A work-group's
// pieces are of different segments and a segment's of different work-groups,
// both in the order of the axis, so g + segment is a number of its own.
__device__ __forceinline__ char *piece_state(const SharedArgs &a, int g, int seg) {
  if (seg < a.groups) return a.ws + static_cast<int64_t>(g + seg) * a.prefix_bytes;
  return a.own_ws + static_cast<int64_t>(g + seg - a.groups) * a.own_bytes;
}

// x of lane `src`.
__device__ __forceinline__ float lane_value(float x, int src) {
  return __int_as_float(__builtin_amdgcn_ds_bpermute(4 * src, __float_as_int(x)));
}

// The arguments again, through a pointer the compiler knows nothing of: read
// where they are used, instead of being held in scalar registers (more than
// there are) across the pieces of a work-group.
typedef const __attribute__((address_space(4))) SharedArgs *args_ptr;
__device__ __forceinline__ args_ptr reread(args_ptr p) {
  asm volatile("" : "+s"(p));
  return p;
}

// Calls piece(args, thread, segment, first page, last page + 1) for the pieces of
// work-group wg, pages counted from the segment's first (uniform over it).
template <typename Piece>
__device__ __forceinline__ void walk_pieces(const SharedArgs &args, int wg, Piece piece) {
  int unit, seg, base;
  {
    const int lane = threadIdx.x & (kWave - 1);
    unit = plan_axis(args, lane, 0).unit;
    const Where at = locate(args, lane, wg * unit);
    seg = at.seg;
    base = at.base;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  for (;; ++seg) {
    // Nothing derived from the lane or the arguments is kept from one piece to
    // the next: hoisted out of this loop it would take the registers the
    // pieces need (three row tiles: 63 of them spilled).
    const SharedArgs &a = (const SharedArgs &)*reread((args_ptr)__builtin_amdgcn_kernarg_segment_ptr());
    const int u0 = wg * unit, u1 = u0 + unit;
    if (seg >= a.groups + a.batch * a.per_seq || base >= u1) return;
    int zero = 0;
    asm volatile("" : "+v"(zero));
    const int tid = wave * kWave + __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, zero));
    const const_i32_ptr lens = (const_i32_ptr)(a.seq_lens);
    const int pages = seg < a.groups ? a.prefix_pages : own_pages(a, lens[(seg - a.groups) / a.per_seq]);
    const int first = base + kPieceCost;  // of the segment's pages on the axis
    base = pages > 0 ? first + pages : base;
    const int s0 = max(u0 - first, 0), s1 = min(u1 - first, pages);
    if (s1 > s0) piece(a, tid, seg, s0, s1);
  }
}

// Pages s0 .. s1 - 1 of segment `seg` (counted from the segment's first page), by
// a work-group of WG_WAVES waves (those behind the first HKV * NWH only keep its barriers).
template <int NT, int HKV, int NWH, bool PH, bool PREFIX, int WG_WAVES = HKV * NWH>
__device__ __forceinline__ void attend_piece(const SharedArgs &a, char *lds_raw, int tid, int wg, int seg, int s0, int s1) {
  constexpr int D = 128;  // PH: dims of a half-head
  using S = Slot<D>;
  using CFG = SplitConfig<D, NT, HKV, NWH, PH>;
  constexpr int RK = CFG::RK, RV = CFG::RV, DQ = CFG::DQ, KSQ = DQ / 64;
  lds_t *lds = (lds_t *)(lds_raw);
  const int lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  if (WG_WAVES > HKV * NWH && wave >= HKV * NWH) {
    __builtin_amdgcn_s_barrier();
    if constexpr (NWH > 1) {
      __syncthreads();
      __syncthreads();
    }
    __syncthreads();
    return;
  }
  const int h = wave % HKV;  // KV head (PH: half-head)
  const int w = wave / HKV;  // position among the NWH waves of this head
  const int hq = PH ? h >> 1 : h;
  const int half = PH ? h & 1 : 0;
  const int n = lane & 15, g = lane >> 4;
  lds_t *qlds = lds + CFG::Q_OFF + hq * CFG::Q_BYTES_PER_HEAD;
  lds_t *kring = lds + wave * CFG::WAVE_BYTES;
  lds_t *vring = kring + RK * S::K_BYTES;
  lds_int *flags = reinterpret_cast<lds_int *>(lds + CFG::FLAG_OFF);
  const LaneOffsets lo = lane_offsets<D, HKV, PH>(a, h, lane);
  const const_i32_ptr lens = (const_i32_ptr)(a.seq_lens);

  const bool shared = PREFIX && seg < a.groups;
  const int os = seg - a.groups;  // own segment
  const int b = shared ? 0 : os / a.per_seq;
  const int sub = shared ? 0 : os - b * a.per_seq;
  const int len = shared ? 0 : lens[b];
  const int p0 = (shared ? 0 : a.prefix_pages) + s0, p1 = (shared ? 0 : a.prefix_pages) + s1;
  const int L0 = shared ? a.prefix_pages * kPage : len;
  const int tok0 = shared ? seg * kGroup : b * a.q_len + sub * kGroup;
  const int ntok = shared ? min(kGroup, a.tokens - tok0) : min(kGroup, a.q_len - sub * kGroup);
  const int rows = ntok * kGqa;
  const int x0 = 2 * p0;
  const int x1 = min(2 * p1, static_cast<int>((static_cast<int64_t>(L0) + 31) / 32));
  const int32_t *bt_row = shared ? a.prefix_table : a.block_table + static_cast<int64_t>(b) * a.bt_stride;

  // Causal ends of this lane's rows: row r is token tok0 + r / 6, of any
  // sequence in a prefix segment.  A row that sees no key at all (a padding
  // sequence) takes no part in the masking, which it would force on every
  // chunk; its state is dropped below.
  WaveState<D, NT> st;
  int far = 0;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = 16 * nt + n;
    int end = L0;
    if (r < rows) {
      const int tok = tok0 + r / kGqa;
      const int sb = tok / a.q_len;
      end = a.seq_lens[sb] - a.q_len + (tok - sb * a.q_len) + 1;
    }
    st.lim[nt] = min(end, L0);
    if (end > 0) far = max(far, kFar - min(st.lim[nt], kFar));
  }
  const int min_end = kFar - wave_max(far);

  const int my0 = x0 + w;
  const int cnt = my0 < x1 ? (x1 - my0 + NWH - 1) / NWH : 0;
  // The query rows' fragments go straight into their operand positions
  // (lane L of fragment (nt, ks) is 16 bytes at 16 L: row 16 nt + n, dims 64
  // ks + 16 g), the rows' scales into the factor words.  The rows behind a
  // short segment's last are other rows of the buffer (it is padded at the
  // end); they are zeroed below.
  int issued = 0;  // DMA bookkeeping as in the decode split kernel
  {
    const int8_t *tile = a.q8 + (hq * a.head_rows + static_cast<int64_t>(tok0) * kGqa) * DQ;
    const float *scales = a.q8_scale + hq * a.head_rows + static_cast<int64_t>(tok0) * kGqa;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (nt % NWH != w) continue;
#pragma unroll
      for (int ks = 2 * half; ks < 2 * half + 2; ++ks) {
        dma16s(tile, static_cast<uint32_t>((16 * nt + n) * DQ + 64 * ks + 16 * g), qlds + (nt * KSQ + ks) * kWave * 16);
        ++issued;
      }
    }
    if (w == 0 && half == 0) {
      if (lane < NT * 16) dma4s(scales, static_cast<uint32_t>(lane * 4), qlds + CFG::Q_FRAG_BYTES);
      ++issued;
    }
  }
  const int q_done = issued;
  // Physical pages of the piece, looked up once (runs of up to 128 pages).
  const bool tab_vgpr = p1 - p0 <= 128;
  int ptab[2] = {-1, -1};
  if (tab_vgpr) {
    int raw[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int p = min(p0 + 64 * i + lane, p1 - 1);
      raw[i] = bt_row[a.ppb <= 1 ? p : p / a.ppb];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int p = p0 + 64 * i + lane;
      const int64_t ph = a.ppb <= 1 ? raw[i] : static_cast<int64_t>(raw[i]) * a.ppb + p % a.ppb;
      ptab[i] = (p < p1 && ph >= 0 && ph < a.num_pages) ? static_cast<int>(ph) : -1;
    }
  }
  auto page_of = [&](int x) -> int {  // x: chunk index in the sequence (wave-uniform)
    const int p = x >> 1;
    if (tab_vgpr) {
      const int d = p - p0;
      const int lo_pg = __builtin_amdgcn_readlane(ptab[0], d & 63);
      const int hi_pg = __builtin_amdgcn_readlane(ptab[1], d & 63);
      return d < 64 ? lo_pg : hi_pg;
    }
    const const_i32_ptr row = (const_i32_ptr)(bt_row);
    const int64_t ph = a.ppb <= 1 ? row[p] : static_cast<int64_t>(row[p / a.ppb]) * a.ppb + p % a.ppb;
    return (ph >= 0 && ph < a.num_pages) ? static_cast<int>(ph) : -1;
  };
  int mk[4] = {0, 0, 0, 0}, mv[4] = {0, 0, 0, 0};
  uint32_t valid_mask = 0;  // bit s: K slot s holds a chunk of a valid page
#pragma unroll
  for (int s = 0; s < (RK > RV ? RK : RV); ++s) {
    if (s >= cnt) break;
    const int xs = my0 + s * NWH;
    if (s < RK) {
      valid_mask |= static_cast<uint32_t>(issue_k<D, HKV>(a, page_of(xs), xs, lo, kring + s * S::K_BYTES)) << s;
      issued += S::NK;
      mk[s] = issued;
    }
    if (s < RV) {
      issue_v<D, HKV, PH>(a, page_of(xs), xs, lo, lane, vring + s * S::V_BYTES);
      issued += S::NVS;
      mv[s] = issued;
    }
  }
  wait_vm(issued - q_done);  // the query rows are here
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (nt % NWH != w || 16 * nt + n < rows) continue;
#pragma unroll
    for (int ks = 2 * half; ks < 2 * half + 2; ++ks)
      *reinterpret_cast<__attribute__((address_space(3))) v4i *>(qlds + ((nt * KSQ + ks) * kWave + lane) * 16) =
          (v4i){0, 0, 0, 0};
  }
  if constexpr (PH) {
    pair_flag_set(flags + wave, 0, lane);
    pair_flag_set(flags + CFG::WAVES + wave, 0, lane);
  } else if constexpr (CFG::BALANCE) {
    pair_flag_set(flags + wave, 0, lane);
  }
  // Fragments and factors visible to both waves of the head (a bare barrier:
  // __syncthreads() would also wait for every ring load in flight).
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float f =
        reinterpret_cast<const __attribute__((address_space(3))) float *>(qlds + CFG::Q_FRAG_BYTES)[nt * 16 + n];
    // Kept above zero so that a masked (-inf) score never meets a zero factor.
    const double c = static_cast<double>(16 * nt + n < rows ? f : 0.f) *
                     (static_cast<double>(kLog2e) / sqrt(static_cast<double>(DQ)));
    st.crow[nt] = fmaxf(static_cast<float>(c), 1e-30f);
    st.lsum[nt] = (v4f){0.f, 0.f, 0.f, 0.f};
    st.corr[nt] = (v4f){0.f, 0.f, 0.f, 0.f};
    st.m_run[nt] = -INFINITY;
    st.thr[nt] = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) st.O[nt][0][j] = (v4f){0.f, 0.f, 0.f, 0.f};
  }

  for (int k = 0; k < cnt; ++k) {
    const int sk = k % RK, sv = k % RV;  // wave-uniform ring slots
    if constexpr (CFG::BALANCE) {
      // The two waves of a SIMD yield to each other (see the decode split kernel).
      pair_flag_set(flags + wave, k, lane);
      const int pk = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const volatile lds_int *>(flags + (wave ^ 4)));
      if (k > pk)
        __builtin_amdgcn_s_setprio(0);
      else
        __builtin_amdgcn_s_setprio(1);
    }
    lds_t *kslot = kring + sk * S::K_BYTES;
    lds_t *vslot = vring + sv * S::V_BYTES;
    int mks = mk[0], mvs = mv[0];
#pragma unroll
    for (int s = 1; s < RK; ++s)
      if (sk == s) mks = mk[s];
#pragma unroll
    for (int s = 1; s < RV; ++s)
      if (sv == s) mvs = mv[s];
    {
      const int left = issued - max(mks, mvs);
      if (left == CFG::STEADY_AFTER)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(CFG::STEADY_AFTER) : "memory");
      else
        wait_vm(left);
    }
    if constexpr (PH) {
      pair_flag_set(flags + wave, k + 1, lane);
      pair_flag_wait(flags + (wave ^ 1), k + 1, lane);
    }
    const bool valid = (valid_mask >> sk) & 1u;
    const int tbase = 32 * (my0 + k * NWH);
    v4i sc[2][NT];
    if constexpr (PH) {
      const lds_t *pslot = lds + (wave ^ 1) * CFG::WAVE_BYTES + sk * S::K_BYTES;
      if (valid) chunk_qk_pair<NT>(half ? pslot : kslot, half ? kslot : pslot, qlds, lane, g, sc);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      pair_flag_set(flags + CFG::WAVES + wave, k + 1, lane);
    } else {
      if (valid) chunk_qk<D, NT>(kslot, qlds, lane, g, sc);
    }
    auto refill_k = [&]() {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      const int xr = my0 + (k + RK) * NWH;
      const uint32_t v = static_cast<uint32_t>(issue_k<D, HKV>(a, page_of(xr), xr, lo, kslot));
      valid_mask = (valid_mask & ~(1u << sk)) | (v << sk);
      issued += S::NK;
#pragma unroll
      for (int s = 0; s < RK; ++s)
        if (sk == s) mk[s] = issued;
    };
    if (CFG::K_EARLY && k + RK < cnt) refill_k();
    if (valid) chunk_softmax_pv<D, NT, PH>(st, sc, vslot, tbase, L0, lane, g, tbase + 32 > min_end);
    if (!CFG::K_EARLY && k + RK < cnt) {
      if constexpr (PH) pair_flag_wait(flags + CFG::WAVES + (wave ^ 1), k + 1, lane);
      refill_k();
    }
    if (k + RV < cnt) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      const int xr = my0 + (k + RV) * NWH;
      issue_v<D, HKV, PH>(a, page_of(xr), xr, lo, lane, vslot);
      issued += S::NVS;
#pragma unroll
      for (int s = 0; s < RV; ++s)
        if (sv == s) mv[s] = issued;
    }
  }

  finalize_output(st);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
    if (st.lim[nt] <= 0) st.m_run[nt] = -INFINITY;

  // The state's form is the decode split kernel's: a quarter of O / l in fp16,
  // then m and l.
  auto write_state = [&]() {
    const int srows = shared ? a.prefix_rows : a.own_rows;
    char *state = piece_state(a, wg, seg);
    _Float16 *obase = reinterpret_cast<_Float16 *>(state);
    float2 *mlbase = reinterpret_cast<float2 *>(state + static_cast<int64_t>(CFG::QHEADS) * srows * DQ * 2);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * nt + 4 * g + i;
        const float m_r = lane_value(st.m_run[nt], 4 * g + i);
        if (r < rows) {
          // A row that saw nothing: zeros, whatever its lanes hold (a padding
          // row's query may be anything).
          const bool seen = m_r != -INFINITY;
          const float l = seen ? st.lsum[nt][i] : 0.f;
          const float f = l > 0.f ? 0.25f / l : 0.f;
          _Float16 *dst = obase + static_cast<int64_t>(hq * srows + r) * DQ + half * 128 + 8 * n;
          v8h o;
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = static_cast<_Float16>(seen ? st.O[nt][0][j][i] * f : 0.f);
          store_wt16(dst, o);
          if (n == 0 && half == 0) store_wt8(mlbase + hq * srows + r, make_float2(m_r, l));
        }
      }
    }
  };
  // Combine the two waves of each head, then write the state.
  if constexpr (NWH > 1) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();  // every ring is drained; the LDS serves the exchange
    float *xb = reinterpret_cast<float *>(lds_raw) + h * (CFG::XCHG_FLOATS);
    if (w == 1) {
      int e = 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        xb[(e++) * kWave + lane] = st.m_run[nt];
#pragma unroll
        for (int i = 0; i < 4; ++i) xb[(e++) * kWave + lane] = st.lsum[nt][i];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) xb[(e++) * kWave + lane] = st.O[nt][0][j][i];
      }
    }
    __syncthreads();
    if (w == 0) {
      int e = 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float m1 = xb[(e++) * kWave + lane];
        const float m0 = st.m_run[nt];
        const float M = fmaxf(m0, m1);
        const float a0 = m0 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m0 - M);
        const float a1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - M);
        st.m_run[nt] = M;
        float a0i[4], a1i[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a0i[i] = lane_value(a0, 4 * g + i);
          a1i[i] = lane_value(a1, 4 * g + i);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) st.lsum[nt][i] = st.lsum[nt][i] * a0i[i] + xb[(e++) * kWave + lane] * a1i[i];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            st.O[nt][0][j][i] = st.O[nt][0][j][i] * a0i[i] + xb[(e++) * kWave + lane] * a1i[i];
          // Combined here, not where the rows are written: there the words
          // of all columns would wait in registers (21 of them spilled).
          asm volatile("" : "+v"(st.O[nt][0][j]));
        }
      }
      write_state();
    }
  }
  if constexpr (NWH == 1) write_state();
  // The next piece's loads overwrite the LDS and count from zero.
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
}

template <int NT, int HKV, int NWH, bool PH>
__global__ __attribute__((amdgpu_flat_work_group_size(64 * HKV * NWH, 64 * HKV * NWH),
                          amdgpu_waves_per_eu(SplitConfig<128, NT, HKV, NWH, PH>::OCC,
                                              SplitConfig<128, NT, HKV, NWH, PH>::OCC)))
void shared_split_kernel(SharedArgs args) {
  __shared__ __attribute__((aligned(16))) char lds[SplitConfig<128, NT, HKV, NWH, PH>::LDS_BYTES];
  const int wg = static_cast<int>(blockIdx.x);
  walk_pieces(args, wg, [&](const SharedArgs &a, int tid, int seg, int s0, int s1) {
    attend_piece<NT, HKV, NWH, PH, true>(a, lds, tid, wg, seg, s0, s1);
  });
}

// ------------------------------------------------------------ many rows
//
// With many query rows the prefix is bound by issue, not by memory: a wave of
// the kernel above spends as much on fetching, unpacking and addressing a
// chunk as on multiplying it.  Here the eight waves of a work-group hold
// consecutive rows of ONE KV head (NT 16-row tiles each) and share every page:
// K stays int8 codes as they are in the cache; V is dequantized once per page
// for all waves, (nibble - zero) * scale / 16 rounded once to fp16 (the 1/16
// keeps rows of the whole fp16 range finite).
//
// Waves w and w + 4 share a SIMD.  They form two groups half a page apart,
// separated by a barrier per phase: in phase A of page p a wave multiplies (O
// += V(p - 1)^T P(p - 1), S = K(p) Q^T) and, between the products, dequantizes
// its share of V(p) (head dim 256: a quarter of it) and issues its share of a
// later page's loads; in phase B it turns S into probabilities and, at head dim
// 256, dequantizes the rest.  So each SIMD holds one wave that feeds the matrix
// core and one that feeds the vector unit; the former issues first (s_setprio),
// as the latter has an instruction for every gap.  With t counting phases, group
// 0 runs A(p) at t = 2p and B(p) at 2p + 1, group 1 one later:
//   raw page p (K codes, V codes): read from t = 2p (A of group 0; at head dim 256
//     group 1, a page ahead in its B, reads its V) to 2p + 1; its V planes, which
//     group 0 loads, are scaled by one wave at t = 2p - 1; the key scales, read
//     to 2p + 2, lie apart.  A wave issues its loads of page p + SLOTS - 1, into
//     the slot of page p - 1, in A(p);
//   V16(p): written at 2p and 2p + 1, read at 2p + 2 and 2p + 3: two buffers.
//
// Bound by issue, the largest calls by power: at head dim 128 a page of a SIMD's
// two waves takes 4,800 cycles, in which its matrix core multiplies for 2,870 (78
// products of 18.4 cycles a wave) and its vector unit works for about 3,300 (48
// exponentials and 240 other instructions a wave).  64 sequences of 4 tokens over
// 1,562 pages run at 2.1 GHz where smaller calls hold 2.4.
// Measured: that call, 4 KV heads, 259 us (the batch op 835): 1,215 TFLOP/s; at a
// large fp16 product's 1,312, and twice that for the int8 one, the two products
// take 180 us.  Head dim 256 459 us, 2 KV heads 137 and 259.  Tried and not
// better: the vector phase first (310 us), no priority (290), row blocks of two
// tiles a wave (4 % at 200 to 256 rows, slower at head dim 256).
// Products are transposed (tokens x rows, dims x rows): a lane owns one row of
// each tile, so the running max, sum and rescale need no exchange but the max
// over the four lanes of a row.
constexpr int kWideWaves = 8;

template <int D>
struct Wide {
  static constexpr int NT = D == 128 ? 3 : 2;    // row tiles a wave holds in registers
  static constexpr int ROWS = kWideWaves * 16 * NT;
  static constexpr int SLOTS = D == 128 ? 4 : 3;
  static constexpr int VROW = D / 2;
  static constexpr int K_BYTES = kPage * D;
  static constexpr int V_OFF = K_BYTES;
  static constexpr int S_OFF = V_OFF + kPage * VROW;   // vs[64] | vz[64]
  static constexpr int SLOT_BYTES = S_OFF + 2 * kPage * 4;
  static constexpr int V16_BYTES = D * kPage * 2;      // [D rows][64 tokens]
  static constexpr int V16_OFF = SLOTS * SLOT_BYTES;
  static constexpr int PAD_OFF = V16_OFF + 2 * V16_BYTES;  // where loads nobody reads land
  // Key scales are read last of a page (D = 256: in B): a ring of their own.
  static constexpr int KS_OFF = PAD_OFF + 256;
  static constexpr int LDS_BYTES = KS_OFF + 4 * kPage * 4;
  static constexpr int KPW = K_BYTES / 1024 / kWideWaves;  // K loads of a wave: 1, 2
  static constexpr int LOADS = KPW + 1 + (D == 128 ? 0 : 1);  // loads of a wave per page
  static_assert(LDS_BYTES <= 163840, "ring exceeds the LDS");
};

// Position of 16-byte chunk c of a V16 row: rows are read 16 at a time at one
// chunk and written 64 at a time at one chunk, both conflict-free.
__device__ __forceinline__ int vswz(int row) { return (row & 7) ^ ((row >> 3) & 1); }

// Pages p0 .. p1 - 1 of the prefix for one row block of one KV head.
template <int D, int HKV>
__device__ __forceinline__ void wide_piece(const SharedArgs &a, char *lds_raw, int tid, int wg, int seg, int p0, int p1) {
  using W = Wide<D>;
  constexpr int NT = W::NT, KS = D / 64, DT = D / 16;
  lds_t *lds = (lds_t *)(lds_raw);
  const int lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int grp = wave >> 2;
  const int n = lane & 15, g = lane >> 4;

  const int h = seg / a.wide_blocks, block = seg - h * a.wide_blocks;
  const int row0 = block * W::ROWS + wave * 16 * NT;  // first row of this wave, of the head's tokens * 6
  const int nrows = a.tokens * kGqa;
  const bool active = row0 < nrows;
  const int pages = p1 - p0;

  // Query rows: lane (n, g) of tile nt holds row 16 nt + n, dims 64 ks + 16 g ...
  // A row behind the batch's last reads the last's length and scale and uses
  // neither, so that all tiles' loads are one round trip.
  v4i qf[NT][KS];
  float crow[NT];
  int lim[NT];
  int far = 0;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = row0 + 16 * nt + n;
    const int64_t at = h * a.head_rows + r;  // the buffer is padded to whole blocks
    const int rl = min(r, nrows - 1), tok = rl / kGqa, sb = tok / a.q_len;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[nt][ks] = *reinterpret_cast<const v4i *>(a.q8 + at * D + 64 * ks + 16 * g);
    crow[nt] = a.q8_scale[h * a.head_rows + rl];
    lim[nt] = a.seq_lens[sb] - a.q_len + (tok - sb * a.q_len) + 1;
  }
  // Physical pages, 64 at a time: lane l holds page p0 + 64 k + l.
  int ptab = -1;
  auto load_table = [&](int k) {
    const int p = min(p0 + 64 * k + lane, p1 - 1);
    const int raw = a.prefix_table[a.ppb <= 1 ? p : p / a.ppb];
    const int64_t ph = a.ppb <= 1 ? raw : static_cast<int64_t>(raw) * a.ppb + p % a.ppb;
    ptab = ph >= 0 && ph < a.num_pages ? static_cast<int>(ph) : -1;
  };
  load_table(0);  // in the query rows' round trip
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const bool live = row0 + 16 * nt + n < nrows;
    if (live && lim[nt] > 0) far = max(far, kFar - min(lim[nt], kFar));
    if (!live) lim[nt] = a.prefix_pages * kPage;
    const double f = live ? static_cast<double>(crow[nt]) : 0.0;
    crow[nt] = fmaxf(static_cast<float>(f * (static_cast<double>(kLog2e) / sqrt(static_cast<double>(D)))), 1e-30f);
  }
  const int min_end = kFar - wave_max(far);

  // The lane for addresses that, kept over the loop, would be what is too many
  // for the registers at head dim 256: formed anew where they are used.
  auto fresh_lane = [&] {
    int l = lane;
    if constexpr (D == 256) asm volatile("" : "+v"(l));
    return l;
  };
  // Lane offsets of this wave's loads of a page: K rows (swizzled as in
  // lane_offsets), V rows, one cell of a plane.
  const int vj = wave & (kPage * W::VROW / 1024 - 1);  // 1 KB piece of V rows
  struct Offsets {
    uint32_t k[W::KPW], v, p;
  };
  auto offsets = [&](int l) {
    Offsets o;
#pragma unroll
    for (int k = 0; k < W::KPW; ++k) {
      constexpr int CPR = D / 16;  // 16-byte chunks of a K row
      const int t = (wave * W::KPW + k) * (1024 / D) + l / CPR;
      o.k[k] = static_cast<uint32_t>(t * (HKV * D) + h * D + 16 * ((l % CPR) ^ kswz<D>(t)));
    }
    o.v = static_cast<uint32_t>((vj * (1024 / W::VROW) + l * 16 / W::VROW) * (HKV * W::VROW) + h * W::VROW + l * 16 % W::VROW);
    o.p = static_cast<uint32_t>((l * HKV + h) * 4);
    return o;
  };
  const Offsets off0 = offsets(lane);
  // Whether page i of the piece is in the cache, for the last SLOTS pages issued.
  uint32_t valid = 0;
  // This wave's loads of page i of the piece (W::LOADS of them, also for a
  // page behind the last or outside the cache, so every page costs the same
  // count): its share of the K rows and of the V rows, and a plane.
  const char *const kbase = reinterpret_cast<const char *>(a.k_cache);
  const char *const vbase = reinterpret_cast<const char *>(a.v_cache);
  // The V planes are loaded by waves of group 0, which waits for a page first.
  const int plane = wave;  // 1: v_scale, 2: v_zero, others k_scale
  const char *const pbase = plane == 1   ? reinterpret_cast<const char *>(a.v_scale)
                            : plane == 2 ? reinterpret_cast<const char *>(a.v_zero)
                                         : reinterpret_cast<const char *>(a.k_scale);
  // Page strides are below 2^31 bytes, page numbers below 2^31.
  const uint32_t k_ps = static_cast<uint32_t>(a.k_ps), v_ps = static_cast<uint32_t>(a.v_ps);
  const uint32_t p_ps = static_cast<uint32_t>(plane == 1 ? a.vs_ps : plane == 2 ? a.vz_ps : a.ks_ps);
  // In three parts, which phase A runs between its products.
  int phys = -1;
  uint32_t ph = 0;
  auto issue_page = [&](int i) __attribute__((always_inline)) {
    if ((i & 63) == 0 && i > 0 && i < pages) load_table(i >> 6);
    phys = i < pages ? __builtin_amdgcn_readlane(ptab, i & 63) : -1;
    const uint32_t bit = 1u << (i % W::SLOTS);
    valid = phys >= 0 ? valid | bit : valid & ~bit;
    ph = static_cast<uint32_t>(max(phys, 0));
  };
  auto issue_k = [&](int i) __attribute__((always_inline)) {
    lds_t *dst = lds + (i % W::SLOTS) * W::SLOT_BYTES;
    const Offsets off = D == 128 ? off0 : offsets(fresh_lane());
#pragma unroll
    for (int k = 0; k < W::KPW; ++k)
      dma16s(kbase + static_cast<uint64_t>(ph) * k_ps, off.k[k], dst + (wave * W::KPW + k) * 1024);
  };
  auto issue_rest = [&](int i) __attribute__((always_inline)) {
    lds_t *dst = lds + (i % W::SLOTS) * W::SLOT_BYTES;
    const Offsets off = D == 128 ? off0 : offsets(fresh_lane());
    if (D == 256 || wave >= 4) dma16s(vbase + static_cast<uint64_t>(ph) * v_ps, off.v, dst + W::V_OFF + vj * 1024);
    if (D == 256 || wave < 4) {
      // D = 128: waves 0 and 3 both fetch k_scale; D = 256: 0 and 3 .. 7.  A page
      // outside the cache holds no keys: its scores are masked in B, and its
      // planes are zeros here, so that its V is zeros whatever page 0 holds.
      lds_t *pdst = plane == 1 || plane == 2 ? dst + W::S_OFF + (plane - 1) * kPage * 4 : lds + W::KS_OFF + (i & 3) * kPage * 4;
      dma4s(pbase + static_cast<uint64_t>(ph) * p_ps, off.p, phys >= 0 ? pdst : lds + W::PAD_OFF);
      if (phys < 0) *reinterpret_cast<__attribute__((address_space(3))) float *>(pdst + 4 * lane) = 0.f;
    }
  };
  auto issue = [&](int i) __attribute__((always_inline)) {
    issue_page(i);
    issue_k(i);
    issue_rest(i);
  };

  v4f O[NT][DT];
  v4f lsum[NT];
  float m_run[NT], thr[NT];
  v4i S[NT][4];
  v8h P[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    lsum[nt] = (v4f){0.f, 0.f, 0.f, 0.f};
    m_run[nt] = -INFINITY;
    thr[nt] = -INFINITY;
#pragma unroll
    for (int j = 0; j < DT; ++j) O[nt][j] = (v4f){0.f, 0.f, 0.f, 0.f};
  }
  const v4i bias = {kScoreBias, kScoreBias, kScoreBias, kScoreBias};
  const v8h ones = {1, 1, 1, 1, 1, 1, 1, 1};

  // The V planes of page i made into what its dequantization takes, by one wave
  // for all: a byte holds two dims, each as fp16 bits n 2^-24 (subnormal, exact),
  // so with s' = 2^20 scale and z' = -zero scale / 16 one fma, rounded once to
  // fp16, gives (n - zero) scale / 16.
  float plane_s, plane_z;
  auto read_planes = [&](int i) __attribute__((always_inline)) {
    const lds_t *planes = lds + (i % W::SLOTS) * W::SLOT_BYTES + W::S_OFF + 4 * lane;
    plane_s = *reinterpret_cast<__attribute__((address_space(3))) const float *>(planes);
    plane_z = *reinterpret_cast<__attribute__((address_space(3))) const float *>(planes + kPage * 4);
  };
  auto scale_planes = [&](int i) __attribute__((always_inline)) {
    if (wave != 0) return;
    lds_t *planes = lds + (i % W::SLOTS) * W::SLOT_BYTES + W::S_OFF + 4 * lane;
    *reinterpret_cast<__attribute__((address_space(3))) float *>(planes) = plane_s * 0x1p20f;
    *reinterpret_cast<__attribute__((address_space(3))) float *>(planes + kPage * 4) = plane_z * (plane_s * -0.0625f);
  };

  // This wave's share of V16(i): tokens 4 wave' + {0..3, 16..19} of its group's
  // 32-token half of the page, byte columns `lane` (D = 256: and 64 + lane).
  // V16 rows are parity * D / 2 + byte column, a lane's eight tokens a 16-byte
  // chunk.
  // In units of one byte column (D = 256: and four tokens, for the registers).
  // All of it in A, at head dim 256 one unit of four (none or two: the same time).
  constexpr int COLS = W::VROW / kWave, TOK = D == 128 ? 8 : 4, UNITS = COLS * 8 / TOK, IN_A = 1;
  typedef _Float16 vth __attribute__((ext_vector_type(TOK)));
  typedef int v2i __attribute__((ext_vector_type(2)));
  v2i bytes;  // of tokens 0 .. 3 | 4 .. 7 of a lane's column
  v4f vs[TOK / 4], vz[TOK / 4];
  vth even, odd;
  auto fetch = [&](int i, int u) __attribute__((always_inline)) {
    const lds_t *raw = lds + (i % W::SLOTS) * W::SLOT_BYTES;
    const int c = u * TOK / 8, e0 = u * TOK % 8 / 4, t0 = 32 * grp + 4 * (wave & 3) + 16 * e0;
    // The transposing read: of 16 lanes, lane 2 j + h reads bytes 8 h .. 8 h + 7 of
    // the sixteen columns in token j, and lane l receives column l of tokens 0 .. 7.
    const int l = fresh_lane(), j = (l & 15) >> 1;
    const int row = 32 * grp + 4 * (wave & 3) + (j & 3) + 16 * (j >> 2);
    bytes = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i *)(
        raw + W::V_OFF + row * W::VROW + c * kWave + 16 * (l >> 4) + 8 * (l & 1)));
    if (e0) bytes[0] = bytes[1];
#pragma unroll
    for (int e = 0; e < TOK / 4; ++e) {
      vs[e] = *reinterpret_cast<__attribute__((address_space(3))) const v4f *>(raw + W::S_OFF + (t0 + 16 * e) * 4);
      vz[e] = *reinterpret_cast<__attribute__((address_space(3))) const v4f *>(raw + W::S_OFF + (kPage + t0 + 16 * e) * 4);
    }
  };
  auto dequantize = [&](int t) __attribute__((always_inline)) {
    // Tokens t and t + 2 of four share a word: the compiler forms each once.
    const uint32_t w = static_cast<uint32_t>(bytes[t >> 2]) >> (8 * (t & 1));
    const v2h lo = __builtin_bit_cast(v2h, w & 0x000F000Fu), hi = __builtin_bit_cast(v2h, (w >> 4) & 0x000F000Fu);
    const float s = vs[t >> 2][t & 3], z = vz[t >> 2][t & 3];
    even[t] = static_cast<_Float16>(fmaf(static_cast<float>(lo[(t >> 1) & 1]), s, z));
    odd[t] = static_cast<_Float16>(fmaf(static_cast<float>(hi[(t >> 1) & 1]), s, z));
  };
  auto put = [&](int i, int u) __attribute__((always_inline)) {
    lds_t *dst = lds + W::V16_OFF + (i & 1) * W::V16_BYTES;
    const int col = u * TOK / 8 * kWave + fresh_lane();
    const int pos = 16 * ((4 * grp + (wave & 3)) ^ vswz(col)) + 2 * (u * TOK % 8);
    *reinterpret_cast<__attribute__((address_space(3))) vth *>(dst + col * 128 + pos) = even;
    *reinterpret_cast<__attribute__((address_space(3))) vth *>(dst + (W::VROW + col) * 128 + pos) = odd;
  };
  auto convert = [&](int i, auto in_a) __attribute__((always_inline)) {
    constexpr int U0 = decltype(in_a)::value ? 0 : IN_A, U1 = decltype(in_a)::value ? IN_A : UNITS;
#pragma unroll
    for (int u = U0; u < U1; ++u) {
      fetch(i, u);
#pragma unroll
      for (int t = 0; t < TOK; ++t) dequantize(t);
      put(i, u);
    }
  };

  // Phase A: O += V(i)^T P and the row sums with it, S = K(i + 1) Q^T, in steps
  // of one operand (16 bytes a lane) and the NT products that use it.  Operands
  // are read AHEAD steps before their use (an LDS round trip takes about as
  // long as eight products), one step's code fenced off from the next.
  constexpr int NV = 2 * DT, NK = 4 * KS, AHEAD = D == 128 ? 6 : 4;
  v4f kscale[4];  // of the page whose scores S holds: tokens 16 ml + 4 g ..
  auto read_kscale = [&](int i) {
#pragma unroll
    for (int ml = 0; ml < 4; ++ml)
      kscale[ml] = *reinterpret_cast<__attribute__((address_space(3))) const v4f *>(
          lds + W::KS_OFF + ((i & 3) * kPage + 16 * ml + 4 * g) * 4);
  };
  auto phase_a = [&](int i, auto with_v) __attribute__((always_inline)) {
    __builtin_amdgcn_s_setprio(1);  // the products first, phase B in their gaps
    constexpr int FIRST = decltype(with_v)::value ? 0 : NV, LAST = NV + NK;
    const lds_t *vsrc = lds + W::V16_OFF + (i & 1) * W::V16_BYTES;
    const lds_t *raw = lds + ((i + 1) % W::SLOTS) * W::SLOT_BYTES;
    auto operand = [&](int x) -> v4i {
      if (x < NV) {
        // Tile j: dims 32 (j / 2) + 2 n' + j % 2 for n' = 0..15, tokens 32 s + ...
        const int s = x / DT, j = x % DT, c = 16 * (j >> 1) + n;
        return *reinterpret_cast<__attribute__((address_space(3))) const v4i *>(
            vsrc + ((j & 1) * W::VROW + c) * 128 + 16 * ((4 * s + g) ^ vswz(c)));
      }
      const int ml = (x - NV) / KS, ks = (x - NV) % KS, t = 16 * ml + n;
      return *reinterpret_cast<__attribute__((address_space(3))) const v4i *>(raw + t * D + 16 * ((4 * ks + g) ^ kswz<D>(t)));
    };
    v4i ring[AHEAD];
#pragma unroll
    for (int x = 0; x < AHEAD; ++x) ring[x] = operand(FIRST + x);
    if constexpr (FIRST != 0) convert(i + 1, std::true_type{});
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (FIRST == 0) {
#pragma unroll
      for (int x = 0; x < NV; ++x) {
        // Between the products, while S is not yet needed: page i + 1 dequantized.
        constexpr int FROM = 3;
        if (x == 1) fetch(i + 1, 0);
        if (x >= FROM && x < FROM + TOK) dequantize(x - FROM);
        if (x == FROM + TOK) put(i + 1, 0);
        const int s = x / DT, j = x % DT;
        const v4i f = ring[x % AHEAD];
        ring[x % AHEAD] = operand(x + AHEAD);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          O[nt][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, f), P[nt][s], O[nt][j], 0, 0, 0);
        if (j == DT - 1) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) lsum[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, P[nt][s], lsum[nt], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int x = NV; x < LAST; ++x) {
      // P's registers are free: a later page's loads, which ahead of the products
      // were 300 (D = 256: 650) cycles without one, and what B needs first.
      if (x == NV) issue_page(i + W::SLOTS);
      if (x == NV + NK / 4) issue_k(i + W::SLOTS);
      if (x == NV + NK / 2) issue_rest(i + W::SLOTS);
      if (D == 128 && x == LAST - 5) read_kscale(i + 1);
      const int k = x - FIRST, ml = (x - NV) / KS, ks = (x - NV) % KS;
      const v4i f = ring[k % AHEAD];
      if (x + AHEAD < LAST) ring[k % AHEAD] = operand(x + AHEAD);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        S[nt][ml] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f, qf[nt][ks], ks ? S[nt][ml] : bias, 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  };
  // P = exp2(score - m - 2) of page i, see chunk_softmax_pv in decode_chunk.h.
  auto softmax = [&](int i, bool there) __attribute__((always_inline)) {
    if constexpr (D == 256) read_kscale(i);
    float t[NT][4][4], mx[NT];
    const int tbase = (p0 + i) * kPage;
    const bool masked = !there || tbase + kPage > min_end;
    const int seen_to = there ? INT32_MAX : 0;
#pragma unroll
    for (int ml = 0; ml < 4; ++ml) {
      const v4f ks = kscale[ml];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float kb = -12582912.0f * ks[e];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) t[nt][ml][e] = fmaf(__int_as_float(S[nt][ml][e]), ks[e], kb);
      }
    }
    if (__builtin_expect(masked, 0)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int ml = 0; ml < 4; ++ml)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (tbase + 16 * ml + 4 * g + e >= min(lim[nt], seen_to)) t[nt][ml][e] = -INFINITY;
    }
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x = -INFINITY;
#pragma unroll
      for (int ml = 0; ml < 4; ++ml)
#pragma unroll
        for (int e = 0; e < 4; ++e) x = fmaxf(x, t[nt][ml][e]);
      mx[nt] = x;
      grow |= x > thr[nt];
    }
    if (__ballot(grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float mnew = fmaxf(m_run[nt], xlane_max16_32(mx[nt]) * crow[nt]);
        const float alpha = m_run[nt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[nt] - mnew);
        m_run[nt] = mnew;
        thr[nt] = (mnew + kRescaleThreshold) / crow[nt];
        lsum[nt] *= alpha;
#pragma unroll
        for (int j = 0; j < DT; ++j) O[nt][j] *= alpha;
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float nm = -fmaxf(m_run[nt], -FLT_MAX) - kPLog2Offset;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          p[e] = __builtin_amdgcn_exp2f(fmaf(t[nt][2 * s + (e >> 2)][e & 3], crow[nt], nm));
        const v2h a0 = pack_h2(p[0], p[1]), a1 = pack_h2(p[2], p[3]), a2 = pack_h2(p[4], p[5]), a3 = pack_h2(p[6], p[7]);
        P[nt][s] = (v8h){a0[0], a0[1], a1[0], a1[1], a2[0], a2[1], a3[0], a3[1]};
      }
    }
  };
  // Ends a phase; with `wait`, `left` pages of this wave's loads may be under way.
  auto end_phase = [&](bool wait, int left) {
    if (wait) {
      if (left == 2)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * W::LOADS) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(W::LOADS) : "memory");
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");  // no LDS access moves over the barrier
    __builtin_amdgcn_sched_barrier(0);
  };

  // The query words are used here, so that the compiler's wait for them does
  // not fall behind the page loads it does not count.
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" ::"v"(qf[nt][ks]));
  // After A(i), in which it issued page i + SLOTS, a wave waits for page i + 2: group
  // 0 (t = 2i + 2) a phase before its V planes are scaled, group 1 (t = 2i + 3) as
  // the page is about to be read.
#pragma unroll
  for (int i = 0; i < W::SLOTS - 1; ++i) issue(i);
  end_phase(true, W::SLOTS - 2);
  read_planes(0);
  scale_planes(0);
  end_phase(false, 0);
  if (grp) {  // group 1 sits out phase 0
    convert(0, std::false_type{});
    end_phase(false, 0);
  }
  auto run = [&](auto compute) {
    constexpr bool C = decltype(compute)::value;
    auto phase = [&](int i, auto with_v) {
      if constexpr (C) {
        phase_a(i, with_v);
      } else {
        issue(i + W::SLOTS);
        convert(i + 1, std::true_type{});
      }
      end_phase(true, W::SLOTS - 2);
    };
    phase(-1, std::false_type{});
    for (int i = 0; i < pages; ++i) {
      read_planes(i + 1);  // group 0's wave 0 scales them; the others read nothing of use
      if constexpr (C) {
        softmax(i, (valid >> (i % W::SLOTS)) & 1u);
        // Used here: its last steps would otherwise be moved over the barrier.
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) asm volatile("" : "+v"(P[nt][0]), "+v"(P[nt][1]));
        __builtin_amdgcn_sched_barrier(0);
      }
      scale_planes(i + 1);
      convert(i + grp, std::false_type{});
      end_phase(false, 0);
      // A(i + 1); behind the last page its scores are of no page and not used.
      phase(i, std::true_type{});
    }
  };
  // Waves whose rows lie behind the batch's only move and dequantize pages.
  if (active)
    run(std::true_type{});
  else
    run(std::false_type{});
  if (!grp) end_phase(false, 0);

  // The state, as in the kernel above: a quarter of O / l (O is a sixteenth),
  // then m and l; lane (n, g) holds dims 32 q + 8 g .. + 7 of row n.
  if (active) {
    char *state = a.ws + static_cast<int64_t>(wg + seg) * a.prefix_bytes;
    float2 *ml = reinterpret_cast<float2 *>(state + static_cast<int64_t>(W::ROWS) * D * 2);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int lr = wave * 16 * NT + 16 * nt + n;
      if (row0 + 16 * nt + n < nrows) {
        const bool seen = lim[nt] > 0 && m_run[nt] != -INFINITY;
        const float l = seen ? lsum[nt][0] : 0.f;
        const float f = l > 0.f ? 4.f / l : 0.f;
        _Float16 *dst = reinterpret_cast<_Float16 *>(state) + static_cast<int64_t>(lr) * D + 8 * g;
#pragma unroll
        for (int q = 0; q < DT / 2; ++q) {
          v8h o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[2 * e] = static_cast<_Float16>(seen ? O[nt][2 * q][e] * f : 0.f);
            o[2 * e + 1] = static_cast<_Float16>(seen ? O[nt][2 * q + 1][e] * f : 0.f);
          }
          store_wt16(dst + 32 * q, o);
        }
        if (g == 0) store_wt8(ml + lr, make_float2(seen ? m_run[nt] : -INFINITY, l));
      }
    }
  }
  // The next piece's loads overwrite the LDS and count from zero.
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
}

// The many-rows form of the whole launch: the prefix's segments (KV heads x row
// blocks) by wide_piece, the sequences' own by attend_piece on the same axis.
template <int D, int HKV, int NT>
__global__ __attribute__((amdgpu_flat_work_group_size(512, 512), amdgpu_waves_per_eu(2, 2)))
void shared_wide_kernel(SharedArgs args) {
  constexpr bool PH = D == 256;
  constexpr int WAVE_HEADS = PH ? 2 * HKV : HKV, NWH = WAVE_HEADS == 8 ? 1 : 2;
  constexpr int OWN_LDS = SplitConfig<128, NT, WAVE_HEADS, NWH, PH>::LDS_BYTES;
  __shared__ __attribute__((aligned(16))) char lds[OWN_LDS > Wide<D>::LDS_BYTES ? OWN_LDS : Wide<D>::LDS_BYTES];
  const int wg = static_cast<int>(blockIdx.x);
  walk_pieces(args, wg, [&](const SharedArgs &a, int tid, int seg, int s0, int s1) {
    if (seg < a.groups)
      wide_piece<D, HKV>(a, lds, tid, wg, seg, s0, s1);
    else
      attend_piece<NT, WAVE_HEADS, NWH, PH, false, kWideWaves>(a, lds, tid, wg, seg, s0, s1);
  });
}

// Folds the states of one column slice of one output row (token, query head):
// the prefix's for its group, then its sequence's own.
template <int D, int TPU>
__global__ __launch_bounds__(TPU) void shared_merge_kernel(SharedArgs a) {
  constexpr int NW = TPU / kWave;
  __shared__ float red[NW * 32 * 10];  // per wave and column: M, l, o[8]
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = threadIdx.x / kWave;
  const int hq = kGqa * a.hkv;
  const int unit = static_cast<int>(blockIdx.x);
  const int row_id = unit / a.merge_cs;
  const int slice = unit - row_id * a.merge_cs;
  const int tok = row_id / hq, qh = row_id - tok * hq;
  const int h = qh / kGqa, i6 = qh - h * kGqa;
  const int b = tok / a.q_len, j = tok - b * a.q_len;

  const int VPR = (D / 8) / a.merge_cs;
  const int SPI = TPU / VPR;
  const int t = threadIdx.x, col = t % VPR, sg = t / VPR;

  const Axis ax = plan_axis(a, lane, b);
  // Pieces of the row's prefix segment and of its own one.
  int pf = 0, pn = 0, of = 0, on = 0;
  const int sub = j / kGroup;
  int ps = tok / kGroup;                                      // prefix segment
  int pr = h * a.prefix_rows + (tok - ps * kGroup) * kGqa + i6;  // the row in its states
  if (a.wide_blocks) {
    const int r = tok * kGqa + i6, block = r / Wide<D>::ROWS;
    ps = h * a.wide_blocks + block;
    pr = r - block * Wide<D>::ROWS;
  }
  const int os = b * a.per_seq + sub;
  if (a.groups) {
    const int first = ps * prefix_cost(a) + kPieceCost;
    pf = first / ax.unit;
    pn = (first + a.prefix_pages - 1) / ax.unit - pf + 1;
  }
  const int len = a.seq_lens[b];
  const int pages = own_pages(a, len);
  if (pages > 0) {
    const int first = a.groups * prefix_cost(a) + ax.before + sub * (pages + kPieceCost) + kPieceCost;
    of = first / ax.unit;
    on = (first + pages - 1) / ax.unit - of + 1;
  }
  const int dcol = 8 * (slice * VPR + col);
  const int orow = h * a.own_rows + (j - sub * kGroup) * kGqa + i6;
  const char *pbase = piece_state(a, pf, ps), *obase = piece_state(a, of, a.groups + os);
  const int64_t p_o = (static_cast<int64_t>(pr) * D + dcol) * 2;
  const int64_t p_ml = static_cast<int64_t>(a.wide_blocks ? 1 : a.hkv) * a.prefix_rows * D * 2 + pr * 8;
  const int64_t o_o = (static_cast<int64_t>(orow) * D + dcol) * 2;
  const int64_t o_ml = static_cast<int64_t>(a.hkv) * a.own_rows * D * 2 + orow * 8;

  MergeAcc acc{-INFINITY, 0.f, (v8f){0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
  const int count = pn + on;
  for (int s0 = sg; s0 < count; s0 += kMergeMU * SPI) {
    // All loads are issued before any is used; a state past the last reads
    // the last one and is dropped.
    MergeRound rd;
    v8h raw[kMergeMU];
    float2 ml[kMergeMU];
#pragma unroll
    for (int u = 0; u < kMergeMU; ++u) {
      const int s = min(s0 + u * SPI, count - 1);
      const bool pre = s < pn;
      const char *state = pre ? pbase + s * a.prefix_bytes : obase + (s - pn) * a.own_bytes;
      ml[u] = *reinterpret_cast<const float2 *>(state + (pre ? p_ml : o_ml));
      raw[u] = *reinterpret_cast<const v8h *>(state + (pre ? p_o : o_o));
    }
#pragma unroll
    for (int u = 0; u < kMergeMU; ++u) {
      const bool live = s0 + u * SPI < count;
      rd.ms[u] = live ? ml[u].x : -INFINITY;
      rd.ls[u] = live ? ml[u].y : 0.f;
      rd.os[u] = live ? __builtin_convertvector(raw[u], v8f) : (v8f){0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    }
    merge_fold_round(acc, rd);
  }
  // The lanes of one column in a wave are col + VPR * k: combine them.
  float Mw = acc.M;
  for (int off = VPR; off < kWave; off <<= 1) Mw = fmaxf(Mw, __shfl_xor(Mw, off, kWave));
  merge_rescale(acc, Mw);
  for (int off = VPR; off < kWave; off <<= 1) {
    acc.l += __shfl_xor(acc.l, off, kWave);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc.o[e] += __shfl_xor(acc.o[e], off, kWave);
  }
  // Then the waves: each publishes its columns, wave 0 folds them.
  if (lane < VPR) {
    float *x = red + (wave * 32 + lane) * 10;
    x[0] = acc.M;
    x[1] = acc.l;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[2 + e] = acc.o[e];
  }
  __syncthreads();
  if (wave != 0 || lane >= VPR) return;
  float Mg = acc.M;
#pragma unroll
  for (int v = 1; v < NW; ++v) Mg = fmaxf(Mg, red[(v * 32 + lane) * 10]);
  merge_rescale(acc, Mg);
#pragma unroll
  for (int v = 1; v < NW; ++v) {
    const float *x = red + (v * 32 + lane) * 10;
    MergeAcc y{x[0], x[1], (v8f){x[2], x[3], x[4], x[5], x[6], x[7], x[8], x[9]}};
    merge_rescale(y, Mg);
    acc.l += y.l;
    acc.o += y.o;
  }
  const float inv = acc.l > 0.f ? 1.f / acc.l : 0.f;
  const int64_t ob = static_cast<int64_t>(tok) * a.out_tok_stride + static_cast<int64_t>(qh) * D + dcol;
  const v8f o = acc.o * inv;
  const uintptr_t addr = reinterpret_cast<uintptr_t>(a.out) + static_cast<uintptr_t>(ob) * (a.out_dtype == K8V4_F32 ? 4 : 2);
  if (a.out_dtype == K8V4_F16 && addr % 16 == 0) {
    *reinterpret_cast<v8h *>(addr) = __builtin_convertvector(o, v8h);
  } else if (a.out_dtype == K8V4_BF16 && addr % 16 == 0) {
    *reinterpret_cast<v8bf *>(addr) = __builtin_convertvector(o, v8bf);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) store_out(a.out, a.out_dtype, ob + e, o[e]);
  }
}

template <int HKV, int NWH, bool PH>
void launch_split(const SharedArgs &a, int tiles, hipStream_t s) {
  const dim3 grid(a.grid), block(64 * HKV * NWH);
  if (tiles == 1)
    shared_split_kernel<1, HKV, NWH, PH><<<grid, block, 0, s>>>(a);
  else if (tiles == 2)
    shared_split_kernel<2, HKV, NWH, PH><<<grid, block, 0, s>>>(a);
  else
    shared_split_kernel<3, HKV, NWH, PH><<<grid, block, 0, s>>>(a);
}

template <int D, int HKV>
void launch_wide(const SharedArgs &a, int tiles, hipStream_t s) {
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

  SharedArgs a;
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
      shared_merge_kernel<128, 64><<<mgrid, dim3(64), 0, s>>>(a);
    else if (tpu == 128)
      shared_merge_kernel<128, 128><<<mgrid, dim3(128), 0, s>>>(a);
    else
      shared_merge_kernel<128, 256><<<mgrid, dim3(256), 0, s>>>(a);
  } else {
    if (tpu == 64)
      shared_merge_kernel<256, 64><<<mgrid, dim3(64), 0, s>>>(a);
    else if (tpu == 128)
      shared_merge_kernel<256, 128><<<mgrid, dim3(128), 0, s>>>(a);
    else
      shared_merge_kernel<256, 256><<<mgrid, dim3(256), 0, s>>>(a);
  }
  return launch_status("k8v4_attn_shared merge");
}
