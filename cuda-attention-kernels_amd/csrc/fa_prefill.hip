// Software-pipelined FlashAttention-2 prefill kernel for MI355X (gfx950).
// (the kernel itself is in fa_prefill_kernel.hpp; shared prefixes use it too)
//
// Serves the reference's dense and varlen prefill, attn_fwd_mma_kernel
// (csrc/flash_attn_mma.cu:63-242) and _attn_fwd_kernel
// (fused_attn/triton_fwd.py:85-172), for 16-bit Q/K/V with D in {16, 32, 64, 128, 256}.
//
// A workgroup of NW waves (8 for D=128 from 4096 queries, 2048 without the causal mask,
// otherwise 4) covers NW*32 queries of one
// q-head; wave w owns 32 of them.  K and V stream through LDS in 64-key tiles (128 at D <= 64,
// 32 at D=256), each in two buffers filled
// straight from memory (buffer_load ... lds).  The product order per wave is the
// same as in the split-K kernel (S^T = K Q^T with the softmax lane-local,
// P^T kept in VGPRs as the B operand of O^T += V^T P^T), but the loop is
// software-pipelined so that one wave always has matrix work and vector work
// that do not depend on each other:
//
//   iteration t:  S_{t+1} = K_{t+1} Q^T            (MFMA)
//                 P_t = 2^(c S_t - m), row sums    (VALU, exp)
//                 O^T += V_t^T P_t^T               (MFMA)
//                 max of S_{t+1}                   (VALU)
//
// MFMA and VALU instructions of one wave overlap when they are interleaved in
// its own instruction stream; a wave that only issues MFMAs while another wave
// of the SIMD only issues VALU work overlaps much less.  K therefore runs one
// tile ahead of V: during iteration t the buffers hold K_{t+1} and V_t while
// K_{t+2} and V_{t+1} are in flight into the other buffers.
//
// Element-wise masking is needed only on the causal diagonal and the key tail; it
// sits behind a uniform branch after the main block, so an iteration is one basic
// block apart from that and the rare online-softmax rescale.
//
// A workgroup's start and end are kept short: the first tiles' DMA goes out before Q
// and before the rest of the set-up, and the output is written through LDS in whole rows.
#include <float.h>

#include <algorithm>

#include <type_traits>

#include "fa_device.hpp"
#include "fa_internal.hpp"
#include "fa_prefill_kernel.hpp"

namespace fa {

// Log-sum-exp merge of the key splits' partials: O = sum_s w_s O_s / sum_s w_s, w_s = 2^(m_s - m) l_s
// (0 when no split saw a key).  A workgroup merges RPT rows of one (batch, q-head) per D/4 threads,
// each thread 4 values of a row, so that consecutive lanes read consecutive 16-byte pieces; the
// loads of CH splits are in flight together.
constexpr int kCombineRows = 2;  // rows per thread

template <int D, class E>
__global__ void __launch_bounds__(256) prefill_combine_kernel(const CombineArgs c) {
  constexpr int TPR = D / 4, RPT = kCombineRows, CH = 4;
  constexpr float NEG_INF = -__builtin_inff();
  const uint32_t rpw = (256 / TPR) * RPT, chunks = ((uint32_t)c.nq + rpw - 1) / rpw;
  const uint32_t bh = blockIdx.x / chunks, chunk = blockIdx.x - bh * chunks;  // b * hq + head
  const uint32_t b = bh / (uint32_t)c.hq, hq = bh - b * (uint32_t)c.hq;
  const int dq = (int)threadIdx.x % TPR, r0 = (int)(chunk * rpw) + (int)threadIdx.x / TPR;
  const int64_t rows = c.rows;
  float m[RPT], l[RPT];
  f32x4 acc[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    m[i] = NEG_INF;
    l[i] = 0.f;
    acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int s0 = 0; s0 < c.n_split; s0 += CH) {
    f32x2 st[CH][RPT];
    f32x4 pv[CH][RPT];
#pragma unroll
    for (int u = 0; u < CH; ++u) {
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const int qi = r0 + i * (256 / TPR);
        st[u][i] = f32x2{NEG_INF, 0.f};
        pv[u][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (s0 + u < c.n_split && qi < c.nq) {
          const int64_t r = (s0 + u) * rows + (int64_t)bh * c.nq + qi;
          st[u][i] = __builtin_bit_cast(f32x2, ld8(c.ml + 2 * r));
          pv[u][i] = __builtin_bit_cast(f32x4, ld16(c.opart + r * D + 4 * dq));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      float mn = m[i];
#pragma unroll
      for (int u = 0; u < CH; ++u) mn = fmaxf(mn, st[u][i][0]);
      const float m_ref = (mn == NEG_INF) ? 0.f : mn;
      const float alpha = fast_exp2(m[i] - m_ref);  // 0 while m = -inf
      l[i] *= alpha;
      acc[i] *= alpha;
#pragma unroll
      for (int u = 0; u < CH; ++u) {
        const float w = fast_exp2(st[u][i][0] - m_ref) * st[u][i][1];
        l[i] += w;
        acc[i] += w * pv[u][i];
      }
      m[i] = mn;
    }
  }
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int qi = r0 + i * (256 / TPR);
    if (qi >= c.nq) continue;
    const float l_safe = (l[i] == 0.f) ? 1.f : l[i];
    const float inv = 1.f / l_safe;
    if (c.lse != nullptr && dq == 0) c.lse[b * c.slb + (int64_t)hq * c.slh + qi] = (m[i] + __log2f(l_safe)) * kLn2;
    uint16_t* o = (uint16_t*)c.o + b * c.sob + (int64_t)hq * c.soh + (int64_t)qi * c.son + 4 * dq;
    st8(o, u32x2{pack2<E>(acc[i][0] * inv, acc[i][1] * inv), pack2<E>(acc[i][2] * inv, acc[i][3] * inv)});
  }
}

template <int D, class E>
static hipError_t launch_prefill_combine(const CombineArgs& c, int64_t heads, hipStream_t stream) {
  constexpr int RPW = 1024 / D * kCombineRows;
  hipLaunchKernelGGL((prefill_combine_kernel<D, E>), dim3((unsigned)(heads * ((c.nq + RPW - 1) / RPW))), dim3(256), 0,
                     stream, c);
  return hipGetLastError();
}

constexpr int kFwdShortTile = 64;  // keys per tile of the three-workgroup form of D=64 and D=32
constexpr int fwd_tile_keys(int d) { return d <= 64 ? 128 : (d == 256 ? 32 : 64); }

template <int D, class E, int NW, bool SPLIT = false, int BN = fwd_tile_keys(D)>
static hipError_t launch_fwd(const TileArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((attn_fwd_kernel<D, E, NW, BN, SPLIT>), dim3((unsigned)a.total), dim3(NW * 64), 0, stream, a);
  return hipGetLastError();
}

template <int D, class E>
static hipError_t launch_fwd_plan(const TileArgs& a, const FwdPlan& plan, hipStream_t stream) {
  if constexpr (D == 128) {
    if (plan.nw == 8) return plan.n_split > 1 ? launch_fwd<D, E, 8, true>(a, stream) : launch_fwd<D, E, 8>(a, stream);
  }
  if (plan.n_split > 1) return launch_fwd<D, E, 4, true>(a, stream);
  if constexpr (D == 64 || D == 32) {
    if (plan.short_tile) return launch_fwd<D, E, 4, false, kFwdShortTile>(a, stream);
  }
  return launch_fwd<D, E, 4>(a, stream);
}

FwdPlan plan_fwd(const fa_fwd_params& p, bool varlen, bool workspace) {
  constexpr int kCus = 256;  // compute units of an MI355X
  const int d = p.head_dim;
  const int nq = varlen ? p.max_seqlen_q : p.seqlen_q, nk = varlen ? p.max_seqlen_k : p.seqlen_k;
  // Dense D=128 with at least 4096 queries (2048 without the causal mask) runs 8 waves (256
  // queries) per workgroup: each K/V tile feeds twice the rows, halving the DMA per MFMA
  // (measured over 4 waves, Hq=32 Hkv=8: +1% causal at N=4096, +2% at 8192 and 16384, +1.7%
  // non-causal at 2048).  Shorter sequences keep 4 (more, shorter workgroups whose start
  // overlaps the other workgroup on the CU: 8 waves lose 5% causal at N=1024, 2.5% at 2048,
  // 0.7% non-causal at 1024).  D=64 keeps 4 (-3% with 8) and D=256 runs one wave per SIMD.
  // Varlen applies the same rule to its longest sequence (max_seqlen_q): a causal batch of 16
  // sequences of 0-4073 tokens keeps 4 waves, and 8 from 2048 measured 2-5% slower on it (its
  // short sequences leave more of a 256-query block empty).  A wave computes the same tiles
  // in the same order with 4 or 8 waves per workgroup, so the result does not depend on the
  // choice.
  FwdPlan plan{};
  plan.nw = (d == 128 && nq >= (p.causal ? 4096 : 2048)) ? 8 : 4;
  plan.n_split = 1;
  // D=64 and D=32 grids beyond two workgroups per CU take 64-key tiles and run three: the extra wave per
  // SIMD hides more, and the last round is shorter.  Up to 512 workgroups, and over more than 4096 keys, the
  // longer tile's iterations are the faster.  GPU time, us, 128-key and 64-key tiles, D=64: B=8 H=16 N=577 28.9 and
  // 25.9 (640 workgroups), B=32 87.6 and 74.6; causal Hq=32 B=8 N=700 40.0 and 35.6, B=4 N=4096 323 and 312, but N=1999
  // (512) 29.6 and 31.8, H=16 N=6000 89.3 and 93.2, B=4 H=8 N=7000 215 and 237.  D=32: B=32 H=16 N=577 64.6 and 56.4,
  // causal Hq=32 B=4 N=4096 236 and 232, B=1 N=8192 207 and 215, N=1999 22.8 and 25.6.  A varlen grid is laid out for
  // its longest sequence and holds fewer workgroups than it counts: it keeps the longer tile (4 sequences up to
  // 1500 tokens, 16 heads, D=64: 28.6 and 37.6).
  plan.short_tile = !varlen && (d == 64 || d == 32) && nk <= 4096 &&
                    (int64_t)p.batch * p.heads_q * ((nq + 127) / 128) > 2 * kCus;

  // Key splits: a call whose row blocks leave compute units idle (few queries against many keys)
  // cuts each block's keys over several workgroups.  The estimate below, in microseconds, charges
  // a CU 1.0 per 128-query tile it runs with two waves per SIMD, 1.15 with one, 0.8 at D=256 (whose
  // workgroups run one per CU); the partials 0.4 per MB (written and read back) and the second
  // launch 10 (4 on the GPU, the rest on the host where Python launches it; the op's native kernel needs about 2).  512 queries against 16384 keys (Hq=32 Hkv=8
  // D=128 causal, 128 row blocks): 223 us unsplit, 132 with 4 splits of 256-query blocks (8
  // splits: 143 with 128-query blocks); 64 queries against 33000: 441 -> 68; 1000 queries against
  // 3000 (256 row blocks) stay unsplit at 52 (2 splits: 58).
  const int64_t heads = (int64_t)p.batch * p.heads_q;
  const int bn = fwd_tile_keys(d);
  if (varlen || !workspace || nk <= 0 || heads * ((nq + 127) / 128) > kCus) return plan;
  const double tiles = (nk + bn - 1) / bn;  // of the last (heaviest) row block
  // mean over the row blocks: a causal first block sees nk - nq + 128 keys
  const double mean = p.causal ? 0.5 * (tiles + std::max(1.0, (double)(nk - nq + 128) / bn)) : tiles;
  auto cost = [&](int nw, int s) {
    const int64_t wgs = heads * ((nq + nw * 32 - 1) / (nw * 32)) * s;
    const double per_cu = (double)((wgs + kCus - 1) / kCus);
    const double tile = d == 256 ? 0.8 : nw == 8 ? 2.0 : per_cu > 1 ? 1.0 : 1.15;
    const double partials = s > 1 ? 10.0 + 0.4e-6 * (double)(heads * nq) * s * d * 4 : 0.0;
    return tile * std::max(tiles, per_cu * mean) / s + partials;
  };
  double best = 0.95 * cost(4, 1);
  for (int nw = 4; nw <= (d == 128 && nq > 128 ? 8 : 4); nw += 4) {
    for (int s = 2; s <= kMaxFwdSplit && s * 4 <= tiles; s *= 2) {
      if (cost(nw, s) < best) {
        best = cost(nw, s);
        plan.nw = nw;
        plan.n_split = s;
      }
    }
  }
  return plan;
}

size_t fwd_workspace_bytes(const fa_fwd_params& p) {
  if (p.dtype != FA_DTYPE_BF16 && p.dtype != FA_DTYPE_F16) return 0;
  const FwdPlan plan = plan_fwd(p, false, true);
  if (plan.n_split <= 1) return 0;
  return (size_t)p.batch * p.heads_q * p.seqlen_q * plan.n_split * ((size_t)p.head_dim + 2) * sizeof(float);
}

fa_status run_fwd(const fa_fwd_params& p, bool varlen, hipStream_t stream, const char** err, void* workspace) {
  const bool mfma = (p.dtype == FA_DTYPE_BF16 || p.dtype == FA_DTYPE_F16) &&
                    (p.head_dim == 16 || p.head_dim == 32 || p.head_dim == 64 || p.head_dim == 128 ||
                     p.head_dim == 256);
  if (p.dtype == FA_DTYPE_F32 && p.head_dim >= 32)
    return run_fwd_f32(p, varlen, stream, err);
  if (!mfma) return run_fwd_generic(p, varlen, stream, err);
  TileArgs a = common_args(p);
  a.o = p.o;
  a.sob = p.o_stride_b;
  a.soh = p.o_stride_h;
  a.son = p.o_stride_n;
  a.o16 = (reinterpret_cast<uintptr_t>(p.o) % 16 == 0 && p.o_stride_h % 8 == 0 && p.o_stride_n % 8 == 0 &&
           (varlen || p.o_stride_b % 8 == 0)) ? 1 : 0;
  a.lse = p.lse;
  a.slb = p.lse_stride_b;
  a.slh = p.lse_stride_h;
  a.varlen = varlen ? 1 : 0;
  if (varlen) {
    a.cu_q = p.cu_seqlens_q;
    a.cu_k = p.cu_seqlens_k;
    a.nq = p.max_seqlen_q;
    a.nk = p.max_seqlen_k;
    a.sqb = a.skb = a.svb = a.sob = a.slb = 0;  // rows are addressed by packed token index
  }
  if (a.nq <= 0 || p.batch <= 0) return FA_OK;
  const FwdPlan plan = plan_fwd(p, varlen, workspace != nullptr);
  const int64_t rows = (int64_t)p.batch * p.heads_q * a.nq;
  if (plan.n_split > 1) {
    a.o = workspace;
    a.ml = (float*)workspace + rows * plan.n_split * p.head_dim;
  }
  a.n_rowblk = (a.nq + plan.nw * 32 - 1) / (plan.nw * 32) * plan.n_split;
  const int64_t kv_groups = (int64_t)p.batch * p.heads_kv;
  // varlen: the (sequence, kv-head) groups are padded to a multiple of the 8 XCDs
  const int64_t groups = varlen ? (kv_groups + 7) / 8 * 8 : kv_groups;
  const int64_t total = groups * a.group * a.n_rowblk;
  if (total > INT32_MAX) {
    *err = "grid too large";
    return FA_ERR_UNSUPPORTED;
  }
  a.total = (int32_t)total;
  a.kv_groups = (int32_t)kv_groups;
  a.n_split = plan.n_split;
  if (!varlen) prefill_schedule(a, p.head_dim, plan.nw);
  hipError_t e = hipErrorInvalidValue;
  const bool bf = p.dtype == FA_DTYPE_BF16;
  switch (p.head_dim) {
    case 128: e = bf ? launch_fwd_plan<128, BF16>(a, plan, stream) : launch_fwd_plan<128, F16>(a, plan, stream); break;
    case 64: e = bf ? launch_fwd_plan<64, BF16>(a, plan, stream) : launch_fwd_plan<64, F16>(a, plan, stream); break;
    case 32: e = bf ? launch_fwd_plan<32, BF16>(a, plan, stream) : launch_fwd_plan<32, F16>(a, plan, stream); break;
    case 16: e = bf ? launch_fwd_plan<16, BF16>(a, plan, stream) : launch_fwd_plan<16, F16>(a, plan, stream); break;
    case 256: e = bf ? launch_fwd_plan<256, BF16>(a, plan, stream) : launch_fwd_plan<256, F16>(a, plan, stream); break;
    default: break;
  }
  if (e != hipSuccess || plan.n_split == 1) return hip_status(e, err);

  const int64_t heads = (int64_t)p.batch * p.heads_q;
  CombineArgs c{};
  c.rows = rows;
  c.opart = (const float*)a.o;
  c.ml = a.ml;
  c.o = p.o;
  c.sob = p.o_stride_b;
  c.soh = p.o_stride_h;
  c.son = p.o_stride_n;
  c.hq = p.heads_q;
  c.nq = p.seqlen_q;
  c.n_split = plan.n_split;
  c.lse = p.lse;
  c.slb = p.lse_stride_b;
  c.slh = p.lse_stride_h;
  switch (p.head_dim) {
    case 128: e = bf ? launch_prefill_combine<128, BF16>(c, heads, stream) : launch_prefill_combine<128, F16>(c, heads, stream); break;
    case 64: e = bf ? launch_prefill_combine<64, BF16>(c, heads, stream) : launch_prefill_combine<64, F16>(c, heads, stream); break;
    case 32: e = bf ? launch_prefill_combine<32, BF16>(c, heads, stream) : launch_prefill_combine<32, F16>(c, heads, stream); break;
    case 16: e = bf ? launch_prefill_combine<16, BF16>(c, heads, stream) : launch_prefill_combine<16, F16>(c, heads, stream); break;
    case 256: e = bf ? launch_prefill_combine<256, BF16>(c, heads, stream) : launch_prefill_combine<256, F16>(c, heads, stream); break;
    default: break;
  }
  return hip_status(e, err);
}

}  // namespace fa
