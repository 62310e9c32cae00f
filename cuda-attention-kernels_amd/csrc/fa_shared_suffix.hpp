// A request's own keys behind the ones that its group shares: one wave's work in attn_fwd_kernel's SHARED form.
//
// The kernel that multiplies a group's rows with the shared keys is bound by the matrix cores and leaves most of the
// memory's bandwidth unused; the requests' own keys are read once for few rows and leave most of the matrix cores unused.
// Both run in one launch, side by side on a compute unit: a workgroup of the latter is four waves that share nothing, each
// with 32 rows (q-heads x queries) of one request and one partition of its keys.
//
// They read at 4-4.5 TB/s behind a start and an end of about 8 us together (alone, 32 requests of 32768 keys and no prefix: 5.9
// TB/s; attention_paged reads those at 6.7).
//
// A wave's 32-key tiles go through its quarter of the workgroup's LDS, K and V in arrays of their own, each refilled as
// soon as it has been read.
#pragma once

#include "fa_device.hpp"
#include "fa_internal.hpp"
#include "fa_shared.hpp"
#include "fa_tile.hpp"

namespace fa {

// Wait until at most N vector-memory instructions of this wave are in flight (they land in order), and order the memory
// accesses around it.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __asm__ volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
  __asm__ volatile("" ::: "memory");
}
// Wait for this wave's LDS reads.
__device__ __forceinline__ void wait_lds() {
  __asm__ volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);
  __asm__ volatile("" ::: "memory");
}

// Lane i's value (uniform i).
__device__ __forceinline__ float lane_value(float x, int i) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), i & 63));
}

// Item `item` of batch x kv-heads x partitions x row blocks.  kl, vl: 64 D bytes each, a tile of 32 keys, or 64 in FP8 (one
// scale block), which stay 8-bit in LDS and are widened as they are read.
template <int D, class E, class KV>
__device__ __forceinline__ void suffix_rows(const SharedTileArgs& a, int item, uint16_t* kl, uint16_t* vl) {
  constexpr bool IS8 = KV::bytes == 1;
  constexpr int KVB = KV::bytes, BN = IS8 ? 64 : 32, KB = BN / 32, KS = D / 16, DB = D / 32;
  constexpr int BLOCKS = BN * D * KVB / 1024;  // 1-KiB loads of a K (or V) tile
  constexpr int ROWS = 1024 / (D * KVB);       // keys of one of them
  constexpr int CPR = D * KVB / 16;            // 16-byte chunks of a row
  constexpr int UNITS = BN / 16;
  constexpr int PG_REGS = 4;
  constexpr float NEG_INF = -__builtin_inff();
  using Shape = typename std::conditional<IS8, TileShape8<D, BN>, TileShape<D, BN>>::type;

  // kv-head innermost: neighbouring waves read the same block-table entries; partitions outermost: those past a short
  // request's end, which have nothing to do, come last
  const SharedArgs& sh = a.shared;
  const int i1 = sh.by_suffix_blocks.of(item), i2 = sh.by_hkv.of(i1), part = sh.by_batch.of(i2);
  const int rb = item - i1 * sh.suffix_blocks, kvh = i1 - i2 * a.hkv, b = i2 - part * a.batch;
  const int prefix = prefix_of_request(a.shared, b), start = shared_keys(a.shared, prefix);
  const int limit = min(prefix + a.shared.max_suffix, a.shared.table_keys);
  const int klo = start + part * a.shared.suffix_split;

  const int lane = (int)threadIdx.x & 63, g = lane >> 5, j = lane & 31;
  const int R = a.group * a.nq, r0 = rb * 32, row = r0 + j;
  const bool row_ok = row < R;
  const int head = row_ok ? sh.by_nq.of(row) : 0;
  const int hq = kvh * a.group + head, qi = row_ok ? row - head * a.nq : 0;

  // block-table entries of the partition (lane i of pg[r] holds entry 64 r + i), then Q, in flight with the length
  const int first_slot = sh.by_page.of(klo);
  int pg[PG_REGS];
  {
    const int end = min(klo + a.shared.suffix_split, limit);
    const int slot_end = end > klo ? sh.by_page.of(end - 1) + 1 : first_slot;
    const int32_t* bt = a.block_table + (int64_t)b * a.sbt;
#pragma unroll
    for (int r = 0; r < PG_REGS; ++r) {
      const int sl = first_slot + 64 * r + lane;
      pg[r] = sl < slot_end ? bt[sl] : -1;
    }
  }
  // a negative scale is applied by negating Q; c stays above 0, so that an excluded score (-inf) times c is -inf
  const uint32_t qsign = a.qk_scale < 0.f ? 0x80008000u : 0u;
  const float c = fmaxf(fabsf(a.qk_scale), kMinScale);
  u32x4 qf[KS];
  {
    const uint16_t* qp = (const uint16_t*)a.q + (int64_t)b * a.sqb + (int64_t)hq * a.sqh + (int64_t)qi * a.sqn + 8 * g;
    const uint32_t keep = row_ok ? 0xffffffffu : 0u;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = (ld16(qp + 16 * s) ^ qsign) & keep;
  }
  const int seq_k = keys_of(a.shared, __builtin_amdgcn_readfirstlane(a.seqlens_k[b]), prefix);
  if (klo >= seq_k) return;  // (the merge does not read this partial)
  __builtin_amdgcn_sched_barrier(0);  // Q's loads stay ahead of the first tile's

  // keys that some row of the wave sees, and from where on not every row does (causal: bottom-right)
  const int offset = seq_k - a.nq;
  int khi = min(seq_k, klo + a.shared.suffix_split), mask_from = khi;
  if (a.causal) {
    const int last = min(r0 + 32, R) - 1;
    const int q0 = r0 - sh.by_nq.of(r0) * a.nq, q1 = last - sh.by_nq.of(last) * a.nq;
    const bool wraps = last + 1 - r0 >= a.nq || q0 > q1;  // (every query is among the rows)
    mask_from = min(khi, (wraps ? 0 : q0) + offset + 1);
    khi = min(khi, (wraps ? a.nq - 1 : q1) + offset + 1);
  }
  const int qlim = a.causal ? qi + offset : seq_k - 1;
  const int n_tiles = khi > klo ? (khi - klo + BN - 1) / BN : 0;

  const uint8_t* kbase = (const uint8_t*)a.k + (int64_t)kvh * a.skh * KVB;
  const uint8_t* vbase = (const uint8_t*)a.v + (int64_t)kvh * a.svh * KVB;
  const int64_t krow = a.skn * KVB, vrow = a.svn * KVB;
  // FP8: lane i holds the scales of the partition's 64-key block i
  float k_scales = 0.f, v_scales = 0.f;
  if constexpr (IS8) {
    const int n = klo + 64 * lane;
    if (n < khi) {
      const int slot = sh.by_page.of(n);
      const int page = a.block_table[(int64_t)b * a.sbt + slot];
      if ((uint32_t)page < (uint32_t)a.num_pages) {  // (keys outside the pool are zeros, with scale 0)
        const int64_t at = (int64_t)page * a.ssb + (int64_t)kvh * a.ssh + (n - slot * a.page_size) / 64;
        k_scales = a.k_scale[at];
        v_scales = a.v_scale[at];
      }
    }
  }
  // 16 keys of a tile lie in one page; keys at or past khi, and pages outside the pool, read as zeros.  (No branches: the
  // selections are a few scalar instructions.)
  struct Rows {
    int page, off, valid;
  };
  auto find = [&](int n0, Rows (&rows)[UNITS]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int n = n0 + 16 * u;
      const int slot = sh.by_page.of(n);
      const int rel = __builtin_amdgcn_readfirstlane(slot - first_slot), ln = rel & 63;
      const int p0 = __builtin_amdgcn_readlane(pg[0], ln), p1 = __builtin_amdgcn_readlane(pg[1], ln),
                p2 = __builtin_amdgcn_readlane(pg[2], ln), p3 = __builtin_amdgcn_readlane(pg[3], ln);
      const int low = rel < 64 ? p0 : p1, high = rel < 192 ? p2 : p3, page = rel < 128 ? low : high;
      const int valid = min(khi - n, 16);
      const bool ok = (valid > 0) & ((uint32_t)page < (uint32_t)a.num_pages);
      rows[u].page = ok ? page : 0;
      rows[u].off = n - slot * a.page_size;
      rows[u].valid = ok ? valid : 0;
    }
  };
  auto load = [&](const Rows (&rows)[UNITS], const uint8_t* base, int64_t page_stride, int64_t row_bytes, uint16_t* dst, bool keys)
      __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const __amdgpu_buffer_rsrc_t rsrc =
          make_rsrc(base + (int64_t)rows[u].page * (page_stride * KVB) + (int64_t)rows[u].off * row_bytes,
                    rows[u].valid > 0 ? (uint32_t)(rows[u].valid - 1) * (uint32_t)row_bytes + (uint32_t)(D * KVB) : 0u);
#pragma unroll
      for (int i = u * BLOCKS / UNITS; i < (u + 1) * BLOCKS / UNITS; ++i) {
        const int r = i * ROWS + lane / CPR, p = lane % CPR;
        const int at = keys ? (kperm(r) & 15) * (int)row_bytes + ((p ^ Shape::swz_k(r)) * 16)
                            : (r & 15) * (int)row_bytes + ((p ^ Shape::swz_v(r)) * 16);
        lds_dma16<true>(rsrc, (uint8_t*)dst + i * 1024, at);
      }
    }
  };

  f32x16 oacc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) oacc[d] = f32x16{};
  float m_run = NEG_INF, l_run = 0.f;
  float v_cur = IS8 ? 0.f : 1.f;  // FP8: O's unit, as in the shared keys' kernel
  // Byte offsets of the operand reads.  K: row j (of a 32-key block), D index 16 s + 8 g; V: transposed reads (ds_read_b64_tr).
  int koffs[KS], voffs[DB][IS8 ? 1 : 2];
#pragma unroll
  for (int s = 0; s < KS; ++s)
    koffs[s] = IS8 ? j * D + ((s ^ Shape::swz_k(j)) * 16) + 8 * g : (j * D + (((2 * s + g) ^ Shape::swz_k(j)) * 8)) * 2;
  const int tr_i = lane & 15, tr_dh = (lane >> 4) & 1;
#pragma unroll
  for (int d = 0; d < DB; ++d) {
#pragma unroll
    for (int hi = 0; hi < (IS8 ? 1 : 2); ++hi) {
      if constexpr (IS8) {
        const int grp = lane >> 4, vr = 8 * (grp >> 1) + (tr_i >> 1);
        voffs[d][hi] = vr * D + (((2 * d + (grp & 1)) ^ Shape::swz_v(vr)) * 16) + 8 * (lane & 1);
      } else {
        const int vr = 8 * g + 4 * hi + (tr_i >> 2), col = 32 * d + 16 * tr_dh + 4 * (tr_i & 3);
        voffs[d][hi] = (vr * D + (((col >> 3) ^ Shape::swz_v(vr)) * 8) + (col & 7)) * 2;
      }
    }
  }

  const uint8_t *k8 = (const uint8_t*)kl, *v8 = (const uint8_t*)vl;
  auto wide = [&](const u32x2& raw) __attribute__((always_inline)) {
    const u32x2 lo = fp8x4_widen<E>(raw[0]), hi = fp8x4_widen<E>(raw[1]);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  Rows next[UNITS];  // where the next tile's rows lie
  if (n_tiles > 0) {
    find(klo, next);
    load(next, kbase, a.spk, krow, kl, true);
    load(next, vbase, a.spv, vrow, vl, false);
    find(klo + BN, next);
  }
  if constexpr (IS8) v_scales = v_units(v_scales);
  for (int t = 0; t < n_tiles; ++t) {
    const int n0 = klo + t * BN;
    wait_loads<BLOCKS>();  // K_t landed; V_t may be in flight
    f32x16 s_acc[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) s_acc[kb] = f32x16{};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const uint8_t* at = k8 + kb * 32 * D * KVB + koffs[s];
        s_acc[kb] = mfma32<E>(IS8 ? wide(ld8(at)) : ld16(at), qf[s], s_acc[kb]);
      }
    }
    const bool more = t + 1 < n_tiles;
    if (more) {
      wait_lds();
      load(next, kbase, a.spk, krow, kl, true);
    }
    float ct = c;
    if constexpr (IS8) ct = fmaxf(c * lane_value(k_scales, t), kMinScale);
    if (n0 + BN > mask_from) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int n = n0 + 32 * kb + 16 * (r >> 3) + 8 * g + (r & 7);
          s_acc[kb][r] = ((n < khi) & (n <= qlim)) ? s_acc[kb][r] : NEG_INF;
        }
      }
    }
    float mt = s_acc[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int r = kb == 0 ? 1 : 0; r < 16; ++r) mt = vmax(mt, s_acc[kb][r]);
    }
    mt = max_xor32(mt * ct);
    // lazy rescale: only when a row's maximum grew by more than 2^8
    const float m_new = vmax(m_run, mt);
    if (__builtin_amdgcn_ballot_w64(m_new > m_run + kRescaleLog2) != 0) {
      const float alpha = fast_exp2(m_run - ((m_new == NEG_INF) ? 0.f : m_new));
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < DB; ++d) oacc[d] *= alpha;
      m_run = m_new;
    }
    float m_safe = (m_run == NEG_INF) ? 0.f : m_run, unfold = 1.f;
    bool valued = true;
    if constexpr (IS8) {  // V's scale: into the exponents, out of the row sum; far from O's unit, O takes it first
      const float vb = lane_value(v_scales, t);
      valued = is_unit(vb);
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
    float rs = 0.f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pf[kb][h][e] = pack2<E>(fast_exp2(__builtin_fmaf(s_acc[kb][8 * h + 2 * e], ct, -m_safe)),
                                  fast_exp2(__builtin_fmaf(s_acc[kb][8 * h + 2 * e + 1], ct, -m_safe)));
          // the row sum of the rounded P that the product takes, so that O / l is a convex combination of V's rows
          rs = sum2<E>(pf[kb][h][e], rs);
        }
      }
    }
    l_run += IS8 ? rs * unfold : rs;
    if constexpr (IS8) {
      if (!valued) {  // the tile has weights, but its values are 0
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) pf[kb][0] = pf[kb][1] = u32x4{0, 0, 0, 0};
      }
    }
    if (more) {
      wait_loads<BLOCKS>();  // V_t landed; K_{t+1} stays in flight
    } else {
      wait_loads<0>();
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* at = v8 + (32 * kb + 16 * h) * D * KVB;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          u32x4 op;
          if constexpr (IS8) {
            op = wide(lds_read_tr8(at + voffs[d][0]));
          } else {
            const u32x2 lo = lds_read_tr16((const uint16_t*)(at + voffs[d][0])), hi = lds_read_tr16((const uint16_t*)(at + voffs[d][1]));
            op = u32x4{lo[0], lo[1], hi[0], hi[1]};
          }
          oacc[d] = mfma32<E>(op, pf[kb][h], oacc[d]);
        }
      }
    }
    if (more) {
      wait_lds();
      load(next, vbase, a.spv, vrow, vl, false);
      find(n0 + 2 * BN, next);
    }
  }

  // the partial: O normalised by its own row sum (zeros without a key), and (m, l)
  const float l_tot = sum_xor32(l_run);
  float inv = l_tot > 0.f ? v_cur / l_tot : 0.f;
  if constexpr (IS8) {
    const int none = first_without_value(v_scales);
    if (none < 64 && klo + 64 * none <= qlim) inv = __builtin_nanf("");
  }
  if (!row_ok) return;
  const int64_t place = ((int64_t)(b * a.hq + hq) * a.nq + qi) * a.shared.part_stride + a.shared.part_base + part;
  float* op = (float*)a.o + place * D + 4 * g;
#pragma unroll
  for (int d = 0; d < DB; ++d) {
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      // (a row without a key here: zeros, whatever V's other rows hold)
      const f32x4 o = {oacc[d][4 * rq] * inv, oacc[d][4 * rq + 1] * inv, oacc[d][4 * rq + 2] * inv, oacc[d][4 * rq + 3] * inv};
      st16(op + d * 32 + 8 * rq, l_tot == 0.f ? u32x4{0, 0, 0, 0} : __builtin_bit_cast(u32x4, o));
    }
  }
  if (g == 0) st8(a.ml + place * 2, __builtin_bit_cast(u32x2, f32x2{m_run, l_tot}));
}

}  // namespace fa
