// The software-pipelined attention kernel of prefill (launched by fa_prefill.hip) and of shared keys (fa_shared.hip).
//
// SHARED: the rows are those of all requests of a group that share their first keys (fa_shared.hpp), K and V lie in pages,
// and the workgroup takes one partition of the shared keys and writes its partial.  The workgroups behind those read the
// requests' own keys (fa_shared_suffix.hpp).
#pragma once

#include <type_traits>

#include "fa_device.hpp"
#include "fa_internal.hpp"
#include "fa_prefill_common.hpp"
#include "fa_shared.hpp"
#include "fa_shared_suffix.hpp"
#include "fa_tile.hpp"

namespace fa {

// Compile-time loop: f(integral_constant<int, I>) for I in [I0, N), always fully unrolled.
template <int I0, int N, class F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (I0 < N) {
    f(std::integral_constant<int, I0>{});
    static_for<I0 + 1, N>(f);
  }
}

template <bool SHARED>
struct FwdArgs {
  using type = typename std::conditional<SHARED, SharedTileArgs, TileArgs>::type;
};

// SPLIT: a.n_split workgroups share a row block's key tiles; each writes an fp32 partial, and
// prefill_combine_kernel merges them (plan_fwd says when).  A kernel of its own: with the split decided
// at run time every call paid for it (GPU time, us, D=64 B=4 H=16 N=130 7.36 -> 7.60, D=128 B=1 Hq=20 Hkv=4
// N=500 13.3 -> 13.7, D=128 not causal B=17 H=16 N=256 24.2 -> 24.9; 238 VGPRs in place of 229).
// Keys per tile (BN): 64 at D=128, 32 at D=256, 128 at D <= 64: 16 KiB per K (or V) tile at D >= 64 and
// 32 MFMAs per iteration; D=32 and D=16 keep 128 keys, whose scores already take 64 registers per lane.
// At D=256 the fp32 output accumulator alone takes 128 registers per lane, so the kernel runs one wave per
// SIMD there.  D=64 and D=32 also come with 64-key tiles, which leave registers and LDS for three
// workgroups per CU in place of two (kFwdShortTile; plan_fwd says when).
template <int D, class E, int NW, int BN, bool SPLIT, bool SHARED = false, class KV = E>
__global__ void __launch_bounds__(NW * 64)
    __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : (D < 128 && BN == 64 && KV::bytes == 2 ? 3 : 2))))
attn_fwd_kernel(const typename FwdArgs<SHARED>::type a) {
  static_assert(NW == 4 || (NW == 8 && D != 256), "4 or 8 waves (two per SIMD) per workgroup");
  // V tiles are at least 32 columns wide, since O^T += V^T P^T works in 32-wide d blocks.  At
  // D=16 the upper 16 columns of a V row in LDS repeat the lower ones (the DMA reads each source
  // chunk twice); they feed only O^T rows 16..31, which are never stored.
  constexpr int DV = D < 32 ? 32 : D;
  using Shape = TileShape<D, BN>;    // K tiles
  using VShape = TileShape<DV, BN>;  // V tiles
  constexpr int TILE = Shape::TILE, VTILE = VShape::TILE;
  constexpr int KB = BN / 32;  // 32-key MFMA blocks per tile
  constexpr int KS = D / 16;   // k-steps of S^T = K Q^T
  constexpr int DB = DV / 32;  // 32-wide d blocks of O^T
  constexpr int QPW = (TILE * 2 / 1024) / NW;    // 1-KiB DMA blocks per wave per K tile
  constexpr int VQPW = (VTILE * 2 / 1024) / NW;  // and per V tile
  static_assert(D == 16 || D == 32 || D == 64 || D == 128 || D == 256, "head dim");
  static_assert((TILE * 2) % (1024 * NW) == 0 && (VTILE * 2) % (1024 * NW) == 0,
                "direct loads must split evenly over the waves");
  constexpr float NEG_INF = -__builtin_inff();
  // FP8 K/V (SHARED): widened on their way into LDS, so that the loop below finds 16-bit tiles
  constexpr bool IS8 = KV::bytes == 1;
  constexpr int KVB = KV::bytes;
  static_assert(!IS8 || SHARED, "FP8 K/V: shared keys only");
  // At D=16 the loop is bound by its vector work (the two products cost 12 MFMAs per 128-key
  // tile against about 200 VALU instructions), so the row sums of P move to the matrix core: one
  // 16x16x32 MFMA per 16-key half-block against a 0/1 operand (rowsum_ones) replaces eight
  // v_dot2 per tile and wave (measured +5.6% at B=4 H=16 N=4096 causal; no gain at D >= 32,
  // and at D=64 the extra registers spill).
  constexpr bool MFMA_ROWSUM = D == 16;

  // Four separate arrays: every access names its buffer at compile time, so the
  // compiler can tell that a DMA into one buffer never aliases reads of another.
  // (SHARED at D=256: room for two of suffix_rows' tiles; one workgroup fits a CU by its registers in any case)
  constexpr int ROOM = SHARED && BN < 64 ? 2 : 1;
  __shared__ __align__(16) uint16_t k_buf0[TILE * ROOM];
  __shared__ __align__(16) uint16_t k_buf1[TILE * ROOM];
  __shared__ __align__(16) uint16_t v_buf0[VTILE * ROOM];
  __shared__ __align__(16) uint16_t v_buf1[VTILE * ROOM];
  if constexpr (SHARED) {
    const int own = (int)blockIdx.x - a.shared.prefix_first;
    if (own >= 0 && own < a.shared.suffix_wgs) {  // the waves of a request's own keys
      const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
      const int item = own * 4 + w, half = (w & 1) * 32 * D;
      if (item >= a.n_items) return;
      // (arrays named at compile time, as above)
      if (w < 2) {
        suffix_rows<D, E, KV>(a, item, k_buf0 + half, v_buf0 + half);
      } else {
        suffix_rows<D, E, KV>(a, item, k_buf1 + half, v_buf1 + half);
      }
      return;
    }
  }

  // ---- work item: (batch, q-head, NW*32-query block) ----------------------------------
  // One scalar load per 64-byte line of the argument block, all issued at entry: left to the
  // compiler, the fields are loaded where they are first used, in four dependent round trips
  // before the first DMA can go out.
  {
    const uint32_t* ap = reinterpret_cast<const uint32_t*>(&a);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(a) / 4); i += 16) {
      const uint32_t x = ap[i];
      __asm__ volatile("" ::"s"(x));
    }
  }
  PrefillItem it;
  int b0 = 0, b1 = 0;     // SHARED: the group's requests,
  int prefix = 0, shared = 0, part = 0;  // its prefix, the shared keys of it, and the workgroup's partition of them
  if constexpr (SHARED) {
    // kv-head innermost (8 of them: one to an XCD, whose L2 then holds its keys), then the row blocks, which read the
    // same keys at about the same time, then the key partitions
    const int item = (int)blockIdx.x < a.shared.prefix_first ? (int)blockIdx.x : (int)blockIdx.x - a.shared.suffix_wgs;
    const int rest = a.shared.by_hkv.of(item);
    it.kvh = item - rest * a.hkv;
    part = a.shared.by_prefix_blocks.of(rest);
    it.rb = rest - part * a.n_rowblk;
    if (!group_of_block(a.shared, a.group * a.nq, NW * 32, it.rb, b0, b1, prefix)) return;  // uniform over the workgroup
    shared = shared_keys(a.shared, prefix);
    if (part * a.shared.prefix_split >= shared) return;
    it.b = b0;  // (the request whose table row is read: below)
    it.hq = it.kvh * a.group;
  } else {
    if (!prefill_item<D>(a, it)) return;  // grid padding (uniform over the workgroup)
  }
  const int b = it.b, hq = it.hq, kvh = it.kvh;
  // SPLIT: a.n_rowblk counts (row block, key split) pairs, the splits of a row block side by side
  const int rb = SPLIT ? it.rb / a.n_split : it.rb;
  const int sp = SPLIT ? it.rb - rb * a.n_split : part;

  int seq_q = a.nq, seq_k = a.nk;
  if constexpr (SHARED) {
    seq_q = (b1 - b0) * a.group * a.nq;  // rows: (request, q-head of the kv-head, query)
    seq_k = shared;
  }
  int64_t qtok0 = 0, ktok0 = 0;
  if (a.varlen) {
    // the offsets are the same for every lane: keep them (and all addresses derived
    // from them) in scalar registers
    const int qs = __builtin_amdgcn_readfirstlane(a.cu_q[b]);
    const int ks = __builtin_amdgcn_readfirstlane(a.cu_k[b]);
    seq_q = __builtin_amdgcn_readfirstlane(a.cu_q[b + 1]) - qs;
    seq_k = __builtin_amdgcn_readfirstlane(a.cu_k[b + 1]) - ks;
    qtok0 = qs;
    ktok0 = ks;
  }
  const int r0 = rb * NW * 32;
  if (r0 >= seq_q) return;  // uniform over the workgroup (zero-length sequences exit here)
  const int offset = seq_k - seq_q;  // bottom-right causal alignment (reference.py:24-33)

  int khi = seq_k;
  if (!SHARED && a.causal) khi = min(khi, min(r0 + NW * 32, seq_q) - 1 + offset + 1);
  int tile0 = 0;  // first tile of this workgroup's key range
  int klo = 0;    // SHARED: its first key
  if constexpr (SHARED) {
    klo = sp * a.shared.prefix_split;
    khi = min(khi, klo + a.shared.prefix_split);
  }
  if constexpr (SPLIT) {
    const int per = ((khi > 0 ? (khi + BN - 1) / BN : 0) + a.n_split - 1) / a.n_split;
    tile0 = sp * per;
    khi = min(khi, (tile0 + per) * BN);
  }

  // ---- lane roles --------------------------------------------------------------------
  const int tid = (int)threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  // Tile t of this workgroup's key range starts at key0(t); local_tiles(n) of the call's first n
  // tiles belong to it or to an earlier split.
  auto key0 = [&](int t) __attribute__((always_inline)) { return SHARED ? klo + t * BN : (tile0 + t) * BN; };
  auto local_tiles = [&](int n) __attribute__((always_inline)) { return SPLIT ? max(n - tile0, 0) : n; };
  int n_tiles = local_tiles(khi > 0 ? (khi + BN - 1) / BN : 0);
  // Tiles [0, n_fast) hold only keys that every query of the workgroup sees (SHARED: of the wave, below).
  const int wg_mask_from = !SHARED && a.causal ? min(khi, r0 + offset + 1) : khi;
  int n_fast = local_tiles(wg_mask_from > 0 ? wg_mask_from / BN : 0);
  const int g = lane >> 5, j = lane & 31;
  const int wr0 = r0 + wave * 32;
  const int qi = wr0 + j;
  const bool row_ok = qi < seq_q;
  const bool wave_active = wr0 < seq_q;
  // keys at or beyond mask_from are not visible to every row of this wave
  int mask_from = khi;
  if (!SHARED && a.causal && wave_active) mask_from = min(khi, wr0 + offset + 1);
  // Key tiles with a key visible to some row of this wave.  Causal: the wave's rows may end
  // before the workgroup's last row, and its later tiles hold only -inf scores (P = 0), so the
  // wave skips their compute and only issues its share of the DMA (with 8 waves up to 3 tiles).
  const int wave_khi = a.causal ? min(khi, min(wr0 + 32, seq_q) - 1 + offset + 1) : khi;
  const int wave_tiles = local_tiles(wave_khi > 0 ? (wave_khi + BN - 1) / BN : 0);
  int qlim = qi + offset;  // last key this lane's row may see (causal)
  // SHARED: row qi's request, q-head and query, and its place in the output
  int bq = b, hrow = hq, nqi = 0, out_row = 0, row_len = 0;
  if constexpr (SHARED) {
    const int in_group = row_ok ? a.shared.by_nq.of(qi) : 0, member = a.shared.by_group.of(in_group);
    nqi = row_ok ? qi - in_group * a.nq : 0;
    bq = b0 + member;
    hrow += in_group - member * a.group;
    out_row = (bq * a.hq + hrow) * a.nq + nqi;
    row_len = a.seqlens_k[bq];
  }

  const uint8_t* kbase = (const uint8_t*)a.k + ((int64_t)b * a.skb + (int64_t)kvh * a.skh + ktok0 * a.skn) * KVB;
  const uint8_t* vbase = (const uint8_t*)a.v + ((int64_t)b * a.svb + (int64_t)kvh * a.svh + ktok0 * a.svn) * KVB;
  const int64_t krow_bytes = a.skn * KVB, vrow_bytes = a.svn * KVB;

  // A negative softmax scale is applied by negating Q (exact for 16-bit floats), so
  // the kernel works with c = |scale| * log2(e) > 0 and max(c*s) = c*max(s).  c is
  // kept away from 0 so that a masked score (-inf) times c stays -inf.
  const uint32_t qsign = a.qk_scale < 0.f ? 0x80008000u : 0u;
  const float c = fmaxf(fabsf(a.qk_scale), kMinScale);

  // ---- Q fragments (B operand of S^T), resident for the whole kernel ----------------
  // (rows past the end read row 0, which exists, and are zeroed).  They are loaded right
  // after the first K/V tiles' DMA is issued, so that both latencies overlap, and fixed up
  // (sign, rows past the end) only once the rest of the set-up is done.
  u32x4 qf[KS];
  auto load_q = [&]() __attribute__((always_inline)) {
    const int64_t qrow = SHARED ? nqi : qtok0 + (row_ok ? qi : 0);
    const uint16_t* qp = (const uint16_t*)a.q + (int64_t)bq * a.sqb + (int64_t)hrow * a.sqh + qrow * a.sqn + 8 * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = ld16(qp + 16 * s);
  };

  // ---- K/V tiles: global -> LDS --------------------------------------------------------
  // Buffer loads past the byte limit return zeros, which zero-fills the keys >= khi of
  // the last tile (masked keys must not carry NaN/Inf into P*V).  The limit fits 32 bits
  // (row stride checked at the C ABI) and is wave-uniform, so descriptors live in SGPRs.
  auto limit = [&](int n0, int64_t row_bytes) __attribute__((always_inline)) {
    const int valid = min(khi - n0, BN);
    return __builtin_amdgcn_readfirstlane(valid > 0 ? (uint32_t)(valid - 1) * (uint32_t)row_bytes + (uint32_t)(D * 2)
                                                    : 0u);
  };
  // SHARED: the rows of a tile that a wave loads lie in one page (16 rows, or 8 of 16; page sizes are multiples of 16, and
  // kperm keeps a row among its 16).  Lane i of pg[r] holds block-table entry 64 r + i of the workgroup's keys.  The address
  // of tile t + 3's rows is formed during iteration t, a few scalar instructions a slot and without a branch: formed in one
  // piece before the first slot it leaves the matrix pipe idle.
  static_assert(!SHARED || (BN / NW <= 16 && QPW == VQPW), "a wave's rows of a tile lie in one page");
  constexpr int PG_REGS = kPrefixPages / 64;
  int pg[PG_REGS] = {};
  const int unit = wave * (BN / NW) / 16 * 16;  // the first of the 16 keys of a tile that hold the wave's rows
  int pslot = 0, poff = 0;                      // their table slot (from the workgroup's first) and offset in the page
  int first_slot = 0, table_row = b;
  if constexpr (SHARED) {
    first_slot = a.shared.by_page.of(klo);
    const int slot_end = a.shared.by_page.of(khi - 1) + 1;
    const int32_t* bt = a.block_table + (int64_t)b * a.sbt;
#pragma unroll
    for (int r = 0; r < PG_REGS; ++r) {
      const int sl = first_slot + 64 * r + lane;
      pg[r] = sl < slot_end ? bt[sl] : -1;
    }
    const int n = klo + unit;
    pslot = a.shared.by_page.of(n);
    poff = n - pslot * a.page_size;
    pslot -= first_slot;
  }
  // SHARED: the table row read above is the group's first request's, which holds the shared keys unless it is shorter (a
  // padded batch): the entries are then loaded again from one that does, or from the longest, whose keys are then all that
  // any row sees.  (Both loads start together.)
  if constexpr (SHARED) {
    int longest;
    table_row = prefix_holder(a.seqlens_k, b0, b1, shared, longest);
    khi = min(khi, longest);
    if (khi <= klo) {  // uniform over the workgroup
      if (row_ok) {
        const int64_t place = (int64_t)out_row * a.shared.part_stride + sp;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) st16((float*)a.o + place * D + g * (D / 2) + 4 * i, u32x4{0, 0, 0, 0});
        if (g == 0) st8(a.ml + place * 2, __builtin_bit_cast(u32x2, f32x2{NEG_INF, 0.f}));
      }
      return;
    }
    n_tiles = (khi - klo + BN - 1) / BN;
    if (table_row != b) {
      const int slot_end = a.shared.by_page.of(khi - 1) + 1;
      const int32_t* bt = a.block_table + (int64_t)table_row * a.sbt;
#pragma unroll
      for (int r = 0; r < PG_REGS; ++r) {
        const int sl = first_slot + 64 * r + lane;
        pg[r] = sl < slot_end ? bt[sl] : -1;
      }
    }
  }
  int step_slots = 0, step_off = 0;
  if constexpr (SHARED) {
    step_slots = a.shared.by_page.of(BN);
    step_off = BN - step_slots * a.page_size;
  }
  struct PageRows {
    const uint8_t* base;
    uint32_t limit;
  };
  PageRows ksrc{}, knew{}, vsrc[3] = {};  // K of tile t + 2 (t + 3), V of tiles t + 1, t + 2 (and t + 3)
  int page_new = 0, valid_new = 0, off_new = 0;
  // in four steps, each a few instructions: the page of tile t's rows, their addresses in K's and in V's pool
  auto source_step = [&](int step, int t) __attribute__((always_inline)) {
    if (step == 0) {
      valid_new = min(khi - (klo + t * BN + unit), 16);
      const int ln = pslot & 63;
      int page = __builtin_amdgcn_readlane(pg[0], ln);
      if constexpr (PG_REGS > 1) {
        const int high = __builtin_amdgcn_readlane(pg[1], ln);
        page = pslot < 64 ? page : high;
      }
      off_new = poff;
      pslot += step_slots;
      poff += step_off;
      const int wrap = poff >= a.page_size ? 1 : 0;
      pslot += wrap;
      poff -= wrap * a.page_size;
      const bool ok = (valid_new > 0) & ((uint32_t)page < (uint32_t)a.num_pages);
      valid_new = ok ? valid_new : 0;
      page_new = ok ? page : 0;
    } else if (step == 1) {
      knew.base = kbase + (int64_t)page_new * (a.spk * KVB);
      knew.limit = valid_new > 0 ? (uint32_t)(valid_new - 1) * (uint32_t)krow_bytes + (uint32_t)(D * KVB) : 0u;
    } else if (step == 2) {
      knew.base += (int64_t)off_new * krow_bytes;
      vsrc[2].base = vbase + (int64_t)page_new * (a.spv * KVB);
    } else {
      vsrc[2].base += (int64_t)off_new * vrow_bytes;
      vsrc[2].limit = valid_new > 0 ? (uint32_t)(valid_new - 1) * (uint32_t)vrow_bytes + (uint32_t)(D * KVB) : 0u;
    }
  };
  auto source_next = [&]() __attribute__((always_inline)) {
    ksrc = knew;
    vsrc[0] = vsrc[1];
    vsrc[1] = vsrc[2];
  };
  // FP8: a wave's rows of a tile come through registers, NP pieces of 16 values a lane, one iteration before they are
  // widened and written to LDS.  The block scales lie in lanes: lane i holds those of the partition's 64-key block i.
  constexpr int NP = IS8 ? BN / NW * D / 1024 : 1;
  u32x4 kreg[NP], vreg[NP];
  float k_scales = 0.f, v_scales = 0.f;
  if constexpr (IS8) {
    const int n = klo + 64 * lane;
    if (n < khi) {
      const int slot = a.shared.by_page.of(n);
      const int page = a.block_table[(int64_t)table_row * a.sbt + slot];
      if ((uint32_t)page < (uint32_t)a.num_pages) {  // (keys outside the pool are zeros, with scale 0)
        const int64_t at = (int64_t)page * a.ssb + (int64_t)kvh * a.ssh + (n - slot * a.page_size) / 64;
        k_scales = a.k_scale[at];
        v_scales = a.v_scale[at];
      }
    }
  }
  auto scale_of = [&](float scales, int t) __attribute__((always_inline)) {
    return lane_value(scales, t * BN / 64);
  };
  // V's rows of tile t, which read as zeros where its scale is no unit of O
  auto valued_rows = [&](PageRows src, int t) __attribute__((always_inline)) {
    src.limit = is_unit(scale_of(v_scales, t)) ? src.limit : 0u;
    return src;
  };
  // what tile t's products are multiplied with to be scores in log2 units
  auto score_scale = [&](int t) __attribute__((always_inline)) { return IS8 ? fmaxf(c * scale_of(k_scales, t), kMinScale) : c; };
  // Lane's row of piece 0, and where piece i lies from there: a uniform distance in memory (the pieces' rows are PR apart,
  // PR a power of two, and kperm moves that bit as a whole), and in LDS a distance and a flip of chunk bits.  The lane's
  // places are formed anew from three registers each time: as registers of their own they would be spilled, and a spill's
  // reload waits for the rows in flight.
  constexpr int PR = IS8 ? 1024 / D : 1;
  int krow0 = 0, vrow0 = 0, col0 = 0;
  if constexpr (IS8 && D == 128) {
    // Eight lanes take half rows of two rows whose swizzles differ in their lowest bit: what they write then differs mod 8
    // chunks (a write goes 128 bytes a cycle, and every second chunk of one row meets each bank twice; 1024 rows x 32768 keys
    // of 8 heads: 162 us, one row after the other 163).
    krow0 = wave * (BN / NW) + 2 * (lane >> 4) + ((lane >> 2) & 1);
    vrow0 = wave * (BN / NW) + (lane >> 4) + 4 * ((lane >> 2) & 1);
    col0 = ((lane & 3) + ((lane >> 1) & 4)) * 16;
  } else if constexpr (IS8) {
    krow0 = vrow0 = wave * (BN / NW) + lane * 16 / D;
    col0 = lane * 16 % D;
  }
  int k_at = (kperm(krow0) & 15) * (int)krow_bytes + col0, v_at = (vrow0 & 15) * (int)vrow_bytes + col0;
  uint32_t k_put = (uint32_t)(krow0 * D + (((col0 / 8) ^ Shape::swz_k(krow0)) * 8)) * 2u;
  uint32_t v_put = (uint32_t)(vrow0 * D + (((col0 / 8) ^ VShape::swz_v(vrow0)) * 8)) * 2u;
  auto fetch = [&](const PageRows& src, int64_t row_bytes, bool keys, int i) __attribute__((always_inline)) {
    int& at = keys ? k_at : v_at;
    __asm__ volatile("" : "+v"(at));
    return buffer_load16<false>(make_rsrc(src.base, src.limit), at + i * (keys ? kperm(PR) : PR) * (int)row_bytes);
  };
  // half h (8 values) of piece i to its place in a tile
  auto widen = [&](const u32x4& piece, uint16_t* dst, bool keys, int i, int h) __attribute__((always_inline)) {
    const u32x2 lo = fp8x4_widen<E>(piece[2 * h]), hi = fp8x4_widen<E>(piece[2 * h + 1]);
    const uint32_t flip = (uint32_t)(h ^ (keys ? Shape::swz_k(i * PR) ^ Shape::swz_k(0) : VShape::swz_v(i * PR) ^ VShape::swz_v(0))) * 16u;
    uint32_t& put = keys ? k_put : v_put;
    __asm__ volatile("" : "+v"(put));
    st16((uint8_t*)dst + ((put ^ flip) + (uint32_t)(i * PR * D * 2)), u32x4{lo[0], lo[1], hi[0], hi[1]});
  };
  // Tile descriptors (a tile past khi gets a zero-length one: its DMA writes zeros) and
  // the wave's i-th 1-KiB DMA instruction of a K or V tile.
  auto k_rsrc = [&](int n0) __attribute__((always_inline)) {
    if constexpr (SHARED) {
      return ksrc;
    } else {
      return make_rsrc(kbase + (int64_t)n0 * krow_bytes, limit(n0, krow_bytes));
    }
  };
  auto v_rsrc = [&](int n0) __attribute__((always_inline)) {
    if constexpr (SHARED) {
      return vsrc[0];
    } else {
      return make_rsrc(vbase + (int64_t)n0 * vrow_bytes, limit(n0, vrow_bytes));
    }
  };
  auto dma_k = [&](const auto& rk, uint16_t* dst, int i) __attribute__((always_inline)) {
    const int blk = wave * QPW + i;
    const int byte = blk * 1024 + lane * 16;
    const int r = byte / (D * 2), p = (byte % (D * 2)) / 16;
    if constexpr (SHARED) {
      lds_dma16<false>(make_rsrc(rk.base, rk.limit), (uint8_t*)dst + blk * 1024,
                       (kperm(r) & 15) * (int)krow_bytes + ((p ^ Shape::swz_k(r)) * 16));
    } else {
      lds_dma16<false>(rk, (uint8_t*)dst + blk * 1024, kperm(r) * (int)krow_bytes + ((p ^ Shape::swz_k(r)) * 16));
    }
  };
  auto dma_v = [&](const auto& rv, uint16_t* dst, int i) __attribute__((always_inline)) {
    const int blk = wave * VQPW + i;
    const int byte = blk * 1024 + lane * 16;
    const int r = byte / (DV * 2), p = (byte % (DV * 2)) / 16;
    int c = p ^ VShape::swz_v(r);
    if constexpr (DV != D) c %= D / 8;  // D=16: the padding chunks re-read their row's chunks
    if constexpr (SHARED) {
      lds_dma16<false>(make_rsrc(rv.base, rv.limit), (uint8_t*)dst + blk * 1024,
                       (r & 15) * (int)vrow_bytes + c * 16);
    } else {
      lds_dma16<false>(rv, (uint8_t*)dst + blk * 1024, r * (int)vrow_bytes + c * 16);
    }
  };
  auto load_k = [&](int n0, uint16_t* dst) __attribute__((always_inline)) {
    const auto rk = k_rsrc(n0);
#pragma unroll
    for (int i = 0; i < QPW; ++i) dma_k(rk, dst, i);
  };
  auto load_v = [&](int n0, uint16_t* dst) __attribute__((always_inline)) {
    const auto rv = v_rsrc(n0);
#pragma unroll
    for (int i = 0; i < VQPW; ++i) dma_v(rv, dst, i);
  };

  // ---- prologue, first half: K_0, V_0, K_1 and then Q go out before the rest of the set-up
  if constexpr (SHARED) {  // (tiles past the last one: no rows)
    auto source = [&](int t) __attribute__((always_inline)) {
      for (int i = 0; i < 4; ++i) source_step(i, t);
      source_next();
    };
    source(0);
    if constexpr (IS8) {
      u32x4 first[NP], second[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) first[i] = fetch(ksrc, krow_bytes, true, i);
#pragma unroll
      for (int i = 0; i < NP; ++i) vreg[i] = fetch(vsrc[1], vrow_bytes, false, i);
      source(1);
#pragma unroll
      for (int i = 0; i < NP; ++i) second[i] = fetch(ksrc, krow_bytes, true, i);
      source(2);
#pragma unroll
      for (int i = 0; i < NP; ++i) kreg[i] = fetch(ksrc, krow_bytes, true, i);
      v_scales = v_units(v_scales);  // (behind the loads above)
#pragma unroll
      for (int i = 0; i < NP; ++i) vreg[i] = is_unit(scale_of(v_scales, 0)) ? vreg[i] : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 2 * NP; ++i) {
        widen(first[i / 2], k_buf0, true, i / 2, i % 2);
        widen(vreg[i / 2], v_buf0, false, i / 2, i % 2);
        widen(second[i / 2], k_buf1, true, i / 2, i % 2);
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) vreg[i] = fetch(valued_rows(vsrc[0], 1), vrow_bytes, false, i);
      source(3);  // (in iteration 0, K of tile 2 and V of tile 1 go to LDS, and K of tile 3 and V of tile 2 are fetched)
    } else {
      load_k(key0(0), k_buf0);
      vsrc[0] = vsrc[1];
      load_v(key0(0), v_buf0);
      source(1);
      load_k(key0(1), k_buf1);
      source(2);  // (in iteration 0: K of tile 2, V of tile 1)
    }
  } else if (n_tiles > 0) {
    load_k(key0(0), k_buf0);
    load_v(key0(0), v_buf0);
    if (n_tiles > 1) load_k(key0(1), k_buf1);
  }
  __builtin_amdgcn_sched_barrier(0);
  load_q();
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (SHARED) {
    // a row sees the shared keys that its request has, up to its own causal end
    const int n = keys_of(a.shared, row_len, prefix);
    qlim = (a.causal ? n - a.nq + nqi : n - 1);
    int least = row_ok ? max(qlim + 1, 0) : khi;
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) least = min(least, __shfl_xor(least, d));
    mask_from = min(khi, __builtin_amdgcn_readfirstlane(least));
    n_fast = mask_from > klo ? (mask_from - klo) / BN : 0;
  }

  // Per-lane LDS byte offsets of the MFMA operand reads.  Unsigned, so that the compiler may
  // fold the buffer bases and the per-slot constants into the ds_read offset field instead of
  // holding one address register per (buffer, slot) pair (16 VGPRs at D=128).
  // K: S^T A-operand, row kb*32 + j, logical chunk 2s + g.
  uint32_t koffs[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) koffs[s] = (uint32_t)(j * D + (((2 * s + g) ^ Shape::swz_k(j)) * 8)) * 2u;
  // V: ds_read_b64_tr_b16 sources, rows 8g + 4*hi + (i >> 2) of each 16-key step,
  // columns 32d + 16dh + 4(i & 3); the row term kb*32 + 16h is a constant offset.
  const int tr_i = lane & 15, tr_dh = (lane >> 4) & 1;
  uint32_t voffs[DB][2];
#pragma unroll
  for (int d = 0; d < DB; ++d) {
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const int vr_row = 8 * g + 4 * hi + (tr_i >> 2);
      const int col = 32 * d + 16 * tr_dh + 4 * (tr_i & 3);
      voffs[d][hi] = (uint32_t)(vr_row * DV + (((col >> 3) ^ VShape::swz_v(vr_row)) * 8) + (col & 7)) * 2u;
    }
  }

  f32x16 oacc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) oacc[d] = f32x16{};
  // running max m_run (log2 domain, scaled) and this lane's share of the row sum
  float m_run = NEG_INF, l_run = 0.f;
  float v_cur = 0.f;  // FP8: O's unit
  f32x4 l_acc = f32x4{};  // MFMA_ROWSUM: every lane's registers hold its own row's full sum
  const u32x4 ones = rowsum_ones<E>(lane);
  // S^T of two consecutive tiles (the loop below is unrolled by 2)
  f32x16 s_a[KB], s_b[KB];

  // ---- building blocks ---------------------------------------------------------------
  auto qk = [&](const uint16_t* Ks, f32x16(&acc)[KB], int s) __attribute__((always_inline)) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      acc[kb] = mfma32<E>(ld16((const uint8_t*)Ks + (kb * 32 * D * 2 + koffs[s])), qf[s], acc[kb]);
  };
  // excluded scores of tile t (keys n0..n0+BN) -> -inf
  auto mask = [&](f32x16(&sc)[KB], int n0) __attribute__((always_inline)) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int n = n0 + kb * 32 + 16 * (r >> 3) + 8 * g + (r & 7);
        const bool ok = (n < khi) & ((!SHARED & (a.causal == 0)) | (n <= qlim));
        sc[kb][r] = ok ? sc[kb][r] : NEG_INF;
      }
    }
  };
  // row max of c*S over the tile (both lanes of the row agree)
  auto tile_max = [&](const f32x16(&sc)[KB], float c) __attribute__((always_inline)) {
    float mx = sc[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int r = (kb == 0 ? 1 : 0); r < 16; ++r) mx = vmax(mx, sc[kb][r]);
    }
    return max_xor32(mx * c);
  };
  // Lazy rescale: keep the running max unless some row of the wave grew by more
  // than 2^8; p = 2^(c*s - m_run) then stays <= 256, and O, l stay consistent
  // because both use the same m_run.
  auto update_max = [&](float mt) __attribute__((always_inline)) {
    const float m_new = vmax(m_run, mt);
    if (__builtin_amdgcn_ballot_w64(m_new > m_run + kRescaleLog2) != 0) {
      const float m_safe_new = (m_new == NEG_INF) ? 0.f : m_new;
      const float alpha = fast_exp2(m_run - m_safe_new);
      if constexpr (MFMA_ROWSUM) {
        l_acc *= alpha;
      } else {
        l_run *= alpha;
      }
#pragma unroll
      for (int d = 0; d < DB; ++d) oacc[d] *= alpha;
      m_run = m_new;
    }
  };
  // One pipelined iteration on tile t: S_{t+1} from K buffer Kn, P_t from cur,
  // O += V_t P_t from V buffer Vc, then the row max of S_{t+1}.  The max is taken
  // unmasked inside the main block and recomputed only when tile t+1 is masked
  // (or does not exist), so the common path is one basic block.
  // The DMA of the next tiles (K_{t+2} into kd, V_{t+1} into vd: buffers every wave has
  // finished reading) is issued one instruction per slot in the first NDMA slots, so every
  // load has the whole iteration to land before the end-of-iteration wait (measured against
  // one instruction every NM / NDMA slots: +1-3% causal N=4096, +2-5% at N=1024).
  auto body = [&](const uint16_t* Kn, const uint16_t* Vc, f32x16(&cur)[KB], f32x16(&nxt)[KB], int t,
                  const auto& rk, uint16_t* kd, const auto& rv, uint16_t* vd)
      __attribute__((always_inline)) {
    // MFMA slots m = 0 .. NQK-1: S_{t+1} (k-step m / KB, key block m % KB);
    // m = NQK .. NM-1: O += V_t P_t (key block, 16-key half, d block; d fastest).
    // The LDS operand of slot m is read PD slots ahead into a ring of registers,
    // so its latency (about two MFMAs) is hidden behind the MFMAs in between; a
    // sched_barrier after every slot keeps this order through scheduling.
    constexpr int NQK = KS * KB, NPV = KB * 2 * DB, NM = NQK + NPV, PD = 3;
    constexpr int NEXP = KB * 8;         // exp micro-steps (2 scores each) for S_t
    constexpr int NMAX = KB * 8;         // max3 steps for S_{t+1}
    // Where the vector work goes.  Exp step u (key block u / 8, 16-key half (u / 4) % 2) runs
    // in S slot u * NQK / ES for u < ES, else in one of the first PVW PV slots, always before
    // the first PV MFMA that reads its P half.  Max steps run in the PV slots from MAX0 on
    // (S_{t+1} is complete two slots after its last MFMA).  At D=128 the exponentials of the
    // second key block move into the first half of the PV slots and the max steps into the
    // second half, so every slot carries about the same vector work against its MFMA (measured
    // against all exponentials in the S slots: +0.5% causal N=4096, +2.1% non-causal N=4096,
    // +1.2% causal N=16384 at Hq=32 Hkv=8; N <= 2048 unchanged).
    constexpr int ES = D == 128 ? NEXP / 2 : NEXP;
    constexpr int PVW = NPV / 2;
    constexpr int MAX0 = D == 128 ? NPV / 2 : 2;
    static_assert(ES % NQK == 0 || NQK % ES == 0, "exp steps must spread evenly over the S slots");
    auto exp_slot = [](int u) constexpr {
      return u < ES ? u * NQK / ES : NQK + (u - ES) * PVW / (NEXP > ES ? NEXP - ES : 1);
    };
    // the first PV slot that reads the P half of exp step u
    auto exp_deadline = [](int u) constexpr { return NQK + ((u / 8) * 2 + (u / 4) % 2) * DB; };
    constexpr int NDMA = QPW + VQPW;
    static_assert(NDMA <= NM, "one DMA instruction per slot");
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) nxt[kb] = f32x16{};
    float m_safe = (m_run == NEG_INF) ? 0.f : m_run;
    // FP8: O is held in units of v_cur, the V block scale of a recent tile.  A tile whose scale vb is within a factor 2 of
    // it takes vb / v_cur into its exponents, and out of its row sum again; any other first brings O to its own scale.
    // (v_scales hold v_units of the scales.)
    const float c_this = score_scale(t), c_next = score_scale(t + 1);
    float unfold = 1.f;
    if constexpr (IS8) {
      const float vb = scale_of(v_scales, t);
      const bool valued = is_unit(vb);  // (else V's rows are zeros)
      if (valued && !(vb <= 2.f * v_cur && v_cur <= 2.f * vb)) {
        const float ratio = v_cur / vb;
#pragma unroll
        for (int d = 0; d < DB; ++d) oacc[d] *= ratio;
        v_cur = vb;
      }
      if (valued) {
        unfold = v_cur / vb;
        m_safe += __log2f(unfold);
      }
    }
    u32x4 pf[KB][2];
    u32x4 opnd[PD + 1];
    float rs = 0.f;
    float mx = NEG_INF;

    auto read = [&](int m) __attribute__((always_inline)) {
      if (m < NQK) {
        const int s = m / KB, kb = m % KB;
        opnd[m % (PD + 1)] = ld16((const uint8_t*)Kn + (kb * 32 * D * 2 + koffs[s]));
      } else {
        const int i = m - NQK, kb = i / (2 * DB), h = (i / DB) % 2, d = i % DB;
        const uint8_t* vp = (const uint8_t*)Vc + (kb * 32 + 16 * h) * DV * 2;
        const u32x2 lo = lds_read_tr16((const uint16_t*)(vp + voffs[d][0]));
        const u32x2 hi = lds_read_tr16((const uint16_t*)(vp + voffs[d][1]));
        opnd[m % (PD + 1)] = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    };
    // exp micro-step u: scores 2e and 2e+1 of chunk (kb, h) of S_t
    auto exp_step = [&](int u) __attribute__((always_inline)) {
      const int kb = u / 8, h = (u / 4) % 2, e = u % 4;
      const float p0 = fast_exp2(__builtin_fmaf(cur[kb][8 * h + 2 * e], c_this, -m_safe));
      const float p1 = fast_exp2(__builtin_fmaf(cur[kb][8 * h + 2 * e + 1], c_this, -m_safe));
      const uint32_t pk = pack2<E>(p0, p1);
      pf[kb][h][e] = pk;
      // the row sum of the rounded P that the MFMA consumes (so O/l is a convex combination)
      if constexpr (!MFMA_ROWSUM) rs = sum2<E>(pk, rs);
    };
    // max step v: scores 2v and 2v+1 of S_{t+1}
    auto max_step = [&](int v) __attribute__((always_inline)) {
      const int kb = v / 8, r = 2 * (v % 8);
      mx = vmax(vmax(mx, nxt[kb][r]), nxt[kb][r + 1]);  // one v_maximum3 per two scores
    };

    // (static_for: every slot index is a compile-time constant, so the operand ring, the
    // accumulator indices and the LDS offsets resolve without relying on loop unrolling)
    static_for<0, PD>([&](auto mc) __attribute__((always_inline)) { read(decltype(mc)::value); });
    static_for<0, NM>([&](auto mc) __attribute__((always_inline)) {
      constexpr int m = decltype(mc)::value;
      if constexpr (m + PD < NM) read(m + PD);
      if constexpr (IS8) {
        // a half of a piece every few slots; the piece's registers then take their next rows
        constexpr int every = NM / (4 * NP);
        if constexpr (m % every == 0 && m / every < 4 * NP) {
          constexpr int u = m / every, i = u / 2 % NP;
          if constexpr (u < 2 * NP) {
            widen(kreg[i], kd, true, i, u % 2);
            if constexpr (u % 2 == 1) kreg[i] = fetch(ksrc, krow_bytes, true, i);
          } else {
            widen(vreg[i], vd, false, i, u % 2);
            if constexpr (u % 2 == 1) vreg[i] = fetch(valued_rows(vsrc[0], t + 2), vrow_bytes, false, i);
          }
        }
      } else if constexpr (m < NDMA) {
        if constexpr (m < QPW) {
          dma_k(rk, kd, m);
        } else {
          dma_v(rv, vd, m - QPW);
        }
      }
      const u32x4 op = opnd[m % (PD + 1)];
      if constexpr (m < NQK) {
        constexpr int s = m / KB, kb = m % KB;
        nxt[kb] = mfma32<E>(op, qf[s], nxt[kb]);
        static_for<0, NEXP>([&](auto uc) __attribute__((always_inline)) {
          constexpr int u = decltype(uc)::value;
          static_assert(exp_slot(u) < exp_deadline(u), "P must be complete before its PV MFMA");
          if constexpr (exp_slot(u) == m) exp_step(u);
        });
      } else {
        constexpr int i = m - NQK, kb = i / (2 * DB), h = (i / DB) % 2, d = i % DB;
        oacc[d] = mfma32<E>(op, pf[kb][h], oacc[d]);
        if constexpr (MFMA_ROWSUM) {
          if constexpr (d == 0) l_acc = mfma16<E>(ones, pf[kb][h], l_acc);  // row sums of 16 keys of P_t
        }
        static_for<0, NEXP>([&](auto uc) __attribute__((always_inline)) {
          constexpr int u = decltype(uc)::value;
          if constexpr (exp_slot(u) == m) exp_step(u);
        });
        if constexpr (i >= MAX0) {
          constexpr int v0 = (i - MAX0) * NMAX / (NPV - MAX0), v1 = (i - MAX0 + 1) * NMAX / (NPV - MAX0);
          static_for<v0, v1>([&](auto vc) __attribute__((always_inline)) { max_step(decltype(vc)::value); });
        }
      }
      if constexpr (SHARED) {
        constexpr int first = NDMA, every = (NM - NDMA) / 4;  // behind this iteration's own loads
        if constexpr (m >= first && (m - first) % every == 0 && (m - first) / every < 4) source_step((m - first) / every, t + (IS8 ? 4 : 3));
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    if constexpr (SHARED) source_next();
    l_run += IS8 ? rs * unfold : rs;
    float mt = max_xor32(mx * c_next);
    if (t + 1 >= n_fast) {
      const int n1 = key0(t + 1);
      if (t + 1 < n_tiles) {
        if (n1 + BN > mask_from) {
          // an empty volatile asm cannot be speculated: without it the compiler
          // if-converts this rare branch and masks every tile in the hot block
          // (measured: ~150 extra VALU/SALU instructions per tile)
          __asm__ volatile("");
          mask(nxt, n1);
          mt = tile_max(nxt, c_next);
        }
      } else {
        mt = NEG_INF;  // past the last tile: nxt holds stale LDS data and is discarded
      }
    }
    update_max(mt);
  };

  // ---- prologue: K_0, V_0, K_1 in flight; S_0 and its max ------------------------------
  {
    const uint32_t keep = row_ok ? 0xffffffffu : 0u;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = (qf[s] ^ qsign) & keep;
  }
  if (n_tiles > 0) {
    lds_dma_wait();
    __syncthreads();
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) s_a[kb] = f32x16{};
#pragma unroll
    for (int s = 0; s < KS; ++s) qk(k_buf0, s_a, s);
    if (key0(0) + BN > mask_from) mask(s_a, key0(0));
    update_max(tile_max(s_a, score_scale(0)));
    __syncthreads();  // every wave has read K_0: its buffer takes K_2
  }

  // ---- main loop, unrolled by 2 so that every buffer is named at compile time --------
  auto step = [&](auto stage_tag, int t) __attribute__((always_inline)) {
    constexpr int ST = decltype(stage_tag)::value;
    uint16_t* k_this = ST == 0 ? k_buf0 : k_buf1;  // held K_t (read already), takes K_{t+2}
    uint16_t* k_next = ST == 0 ? k_buf1 : k_buf0;  // holds K_{t+1}
    uint16_t* v_this = ST == 0 ? v_buf0 : v_buf1;  // holds V_t
    uint16_t* v_next = ST == 0 ? v_buf1 : v_buf0;  // takes V_{t+1}
    auto& cur = ST == 0 ? s_a : s_b;
    auto& nxt = ST == 0 ? s_b : s_a;
    // K_{t+2} and V_{t+1} (zero-length descriptors past the last tile)
    if (NW == 4 || t < wave_tiles) {
      body(k_next, v_this, cur, nxt, t, k_rsrc(key0(t + 2)), k_this, v_rsrc(key0(t + 1)), v_next);
    } else {
      const auto rk = k_rsrc(key0(t + 2)), rv = v_rsrc(key0(t + 1));
#pragma unroll
      for (int i = 0; i < QPW; ++i) dma_k(rk, k_this, i);
#pragma unroll
      for (int i = 0; i < VQPW; ++i) dma_v(rv, v_next, i);
    }
    if constexpr (IS8) {
      // what is in flight goes to registers: only the writes to LDS, and the reads of it, have to be done
      __asm__ volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    } else {
      lds_dma_wait();
      __syncthreads();
    }
  };
  for (int t = 0; t < n_tiles; t += 2) {
    step(std::integral_constant<int, 0>{}, t);
    if (t + 1 < n_tiles) step(std::integral_constant<int, 1>{}, t + 1);
  }

  // ---- epilogue ------------------------------------------------------------------------
  // Every wave has passed the last tile's barrier and its DMA has landed, so the K/V buffers are
  // free for staging the output.
  if (!wave_active) return;
  // each lane summed its 16 of the row's keys per tile (or holds the full sum, MFMA_ROWSUM)
  const float l_tot = MFMA_ROWSUM ? l_acc[0] : sum_xor32(l_run);
  if constexpr (SPLIT || SHARED) {
    // SHARED: every output row has part_stride places for partials
    int part_stride = 0;
    if constexpr (SHARED) part_stride = a.shared.part_stride;
    // fp32 partial of key split sp: O normalised by its own row sum (zeros for a row without keys
    // here) and (m, l), [S][B, Hq, Nq][D]
    const int64_t rows = (int64_t)a.kv_groups * a.group * seq_q;
    const int64_t row0 = sp * rows + ((int64_t)b * a.hq + hq) * seq_q + wr0;
    float inv = l_tot > 0.f ? (IS8 ? v_cur : 1.f) / l_tot : 0.f;
    if constexpr (SHARED) {  // (a row without a key here: zeros, whatever V's other rows hold)
#pragma unroll
      for (int d = 0; d < DB; ++d) {
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[d][r] = l_tot == 0.f ? 0.f : oacc[d][r];
      }
      if constexpr (IS8) {
        const int none = first_without_value(v_scales);
        if (none < 64 && klo + 64 * none <= qlim) inv = __builtin_nanf("");
      }
    }
    if (row_ok && g == 0) st8(a.ml + (SHARED ? (int64_t)out_row * part_stride + sp : row0 + j) * 2, __builtin_bit_cast(u32x2, f32x2{m_run, l_tot}));
    if constexpr (NW * 32 * D * 4 <= 4 * TILE * 2) {
      // through LDS, as the output below: whole rows per store instruction
      constexpr int NCH = D / 4, REG = 32 * D * 4 / 2, PER_BUF = TILE / REG;
      const int bi = wave / PER_BUF;
      float* stage = (float*)((bi == 0 ? k_buf0 : bi == 1 ? k_buf1 : bi == 2 ? v_buf0 : v_buf1) + (wave % PER_BUF) * REG);
#pragma unroll
      for (int d = 0; d < DB; ++d) {
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
          if (d * 32 + 8 * rq >= D) continue;
          const int c = 8 * d + 2 * rq + g;
          *(f32x4*)(stage + j * D + ((c ^ (j & (NCH - 1))) * 4)) = f32x4{oacc[d][4 * rq] * inv, oacc[d][4 * rq + 1] * inv,
                                                                         oacc[d][4 * rq + 2] * inv, oacc[d][4 * rq + 3] * inv};
        }
      }
      constexpr int RPI = 64 / NCH;  // rows per 64-lane read
      const int cc = lane % NCH;
#pragma unroll
      for (int i = 0; i < 32 / RPI; ++i) {
        const int r = i * RPI + lane / NCH;
        const u32x4 v = ld16(stage + r * D + ((cc ^ (r & (NCH - 1))) * 4));
        if constexpr (SHARED) {
          const int64_t at = (int64_t)__shfl(out_row, r) * part_stride + sp;
          if (wr0 + r < seq_q) st16((float*)a.o + at * D + cc * 4, v);
        } else {
          if (wr0 + r < seq_q) st16((float*)a.o + (row0 + r) * D + cc * 4, v);
        }
      }
    } else if (row_ok) {
      float* op = (float*)a.o + (SHARED ? (int64_t)out_row * part_stride + sp : row0 + j) * D;
#pragma unroll
      for (int d = 0; d < DB; ++d) {
#pragma unroll
        for (int rq = 0; rq < 4; ++rq)
          st16(op + d * 32 + 8 * rq + 4 * g, __builtin_bit_cast(u32x4, f32x4{oacc[d][4 * rq] * inv, oacc[d][4 * rq + 1] * inv,
                                                                          oacc[d][4 * rq + 2] * inv, oacc[d][4 * rq + 3] * inv}));
      }
    }
    return;
  }
  // Rows that saw no key have l == 0 and emit zeros (triton_fwd.py:163-165).
  const float l_safe = (l_tot == 0.f) ? 1.f : l_tot;
  const float inv = 1.f / l_safe;
  // O is staged through LDS, row-major with 16-byte chunks XOR-swizzled by row, and written
  // back in whole rows: a lane of the O^T fragment holds 4 values of each of 16 chunks of one
  // row, so storing from the fragment sends each instruction to 32 rows (32 partial cache
  // lines); from LDS, 16 consecutive lanes write one row's 256 bytes (D=128).  Each wave takes its
  // own 32*D-element region of the K/V buffers.
  {
    constexpr int NCH = D / 8;                       // 16-byte chunks per row
    constexpr int SWZ = NCH < 16 ? NCH - 1 : 15;     // chunk swizzle by row
    constexpr int REG = 32 * D;                      // elements per wave
    constexpr int PER_BUF = TILE / REG;              // wave regions per buffer
    static_assert(PER_BUF >= 1 && VTILE >= TILE && NW <= 4 * PER_BUF, "O staging must fit the K/V buffers");
    const int bi = wave / PER_BUF;
    uint16_t* stage = (bi == 0 ? k_buf0 : bi == 1 ? k_buf1 : bi == 2 ? v_buf0 : v_buf1) + (wave % PER_BUF) * REG;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        if (d * 32 + 8 * rq >= D) continue;  // D=16: O^T rows 16..31 are padding
        const int c = 4 * d + rq;            // chunk of d values d*32 + 8*rq .. +7; this lane holds half g
        *reinterpret_cast<u32x2*>(stage + j * D + ((c ^ (j & SWZ)) * 8) + 4 * g) =
            u32x2{pack2<E>(oacc[d][4 * rq] * inv, oacc[d][4 * rq + 1] * inv),
                  pack2<E>(oacc[d][4 * rq + 2] * inv, oacc[d][4 * rq + 3] * inv)};
      }
    }
    constexpr int RPI = 64 / NCH;  // rows per 64-lane read
    const int cc = lane % NCH;
    uint16_t* obase = (uint16_t*)a.o + (int64_t)b * a.sob + (int64_t)hq * a.soh + (qtok0 + wr0) * a.son;
#pragma unroll
    for (int i = 0; i < 32 / RPI; ++i) {
      const int r = i * RPI + lane / NCH;
      const u32x4 v = *reinterpret_cast<const u32x4*>(stage + r * D + ((cc ^ (r & SWZ)) * 8));
      if (wr0 + r < seq_q) {
        uint16_t* dst = obase + (int64_t)r * a.son + cc * 8;
        if (a.o16) {
          st16(dst, v);
        } else {
          st8(dst, u32x2{v[0], v[1]});
          st8(dst + 4, u32x2{v[2], v[3]});
        }
      }
    }
  }
  if (row_ok && a.lse != nullptr && g == 0) {
    // natural-log LSE (triton_fwd.py:169-172)
    a.lse[(int64_t)b * a.slb + (int64_t)hq * a.slh + (qtok0 + qi)] = (m_run + __log2f(l_safe)) * kLn2;
  }
}

}  // namespace fa
