// Attention over a 4-bit K/V cache, and attention that scores the keys of its cache (4-bit or 16-bit).
//
// For queries q_r (the G * n_q (q-head, query) rows that share a kv-head) and keys j of the first seqlens_k[b]:
//   K_j = ks_j kc_j + kz_j,  V_j = vs_j vc_j + vz_j        (kc, vc: D codes of 4 bits; one fp16 pair a row)
//   s_rj = c q_r . K_j,  p_rj = 2^(s_rj - m_r),  o_r = sum_j p_rj V_j / sum_j p_rj     (c = scale * log2 e)
//   score_j = sum_r p_rj / sum_j' p_rj'                                               (attention_scored)
//
// Decomposition.  Keys are cut into partitions of split_len; a workgroup of four waves takes one partition of one
// (batch, kv-head) for up to 16 * RT rows, its waves every fourth 32-key tile each; the waves' (m, l, O) are merged
// through LDS into one fp32 partial, and splitk_combine_kernel merges the partitions.  Bound by the bytes of the
// cache: D + 8 a key at 4 bits, 4 D at 16.
//
// No K or V goes through LDS: with v_mfma_f32_16x16x32 every operand is a lane's own load.
//   S^T = K Q^T      A: lane (r = l % 16, g = l / 16) holds 8 channels of one key as it lies in memory.  The channels'
//                    order along the contraction is free, as Q is loaded in the same order.
//   P^T              C: lane (column = row of Q, g) holds rows 4g..4g+3 of two 16-key blocks.  Block t, row 4a + i is
//                    made key 8a + 4t + i of the tile, so that a lane's eight scores are keys 8g .. 8g+7:
//                    the B operand of the next product, in place.
//   O^T += V^T P^T   A: lane (r, g) needs keys 8g..8g+7 of one channel.  It loads D/16 channels of each of those keys
//                    and pairs two keys' codes (or halves) with v_perm; the n-th product takes its n-th channel.
//
// Codes become bf16 (Q fp16: fp16, for K) as 1 + code/16: the code is shifted to the top of the mantissa and the
// exponent of 1 is or-ed in, two codes an instruction pair.  The product with K starts from -sum(q) so that it is
// q . kc / 16 (the 1s cancel against values of their own size: no precision is lost to them), and
//   s = (16 c ks) (q . kc/16) + (c kz) sum(q).
// V's scale goes into P, rounded to bf16 (an fp16 product could leave fp16's range: vs is as small as V is), and the
// sum of what was rounded takes the mean of the 1s and codes out again:
//   o = sum_j P'_j (1 + vc_j/16) - (1 + 7.5/16) sum_j P'_j + sum_j p_j (vz_j + 7.5 vs_j),   P'_j = bf16(16 vs_j p_j)
// so that P's rounding (2^-8 of itself) meets only (code - 7.5)/16, at most 0.47 of it.  Everything else is fp32.
//
// Scores.  p needs the row's final sum, which no partition has.  The s of a row and key are written as they are
// (4 bytes: 6% of a 16-bit key's bytes at D=128 and four rows, 12% of a 4-bit one's), and score_finish_kernel turns them into
// weights once the combine has written the rows' log-sum-exp.  A second pass over K would read half the cache again.
#include <algorithm>

#include "fa_device.hpp"
#include "fa_internal.hpp"

namespace fa {

namespace {

constexpr int kCacheWaves = 4;
constexpr int kTile = 32;         // keys a wave step
constexpr int kMaxSlots = 258;    // block-table entries of a partition (paged)

__device__ __forceinline__ float max_xor16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x),
                                                  false, false);
  return vmax(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float sum_xor16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x),
                                                  false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}
// over the four lanes of a column
__device__ __forceinline__ float max_groups(float x) { return max_xor32(max_xor16(x)); }
__device__ __forceinline__ float sum_groups(float x) { return sum_xor32(sum_xor16(x)); }

// Nibble n (0..3) of both halves of x as two 16-bit floats 1 + code/16.
template <class E, int N>
__device__ __forceinline__ uint32_t codes2(uint32_t x) {
  constexpr int at = std::is_same<E, BF16>::value ? 3 : 6;  // the top four bits of the mantissa
  constexpr uint32_t mask = (0xfu << at) * 0x10001u, one = std::is_same<E, BF16>::value ? 0x3f803f80u : 0x3c003c00u;
  constexpr int sh = 4 * N - at;
  const uint32_t y = sh >= 0 ? x >> (sh & 31) : x << ((-sh) & 31);
  return (y & mask) | one;
}

// halves {a.lo, b.lo} and {a.hi, b.hi}
__device__ __forceinline__ uint32_t pair_lo(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t pair_hi(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

template <int W>
struct Words {
  uint32_t w[W];
};

// W words (W = 0: one 16-bit half) of a buffer, or of memory
template <int W>
__device__ __forceinline__ void buffer_words(__amdgpu_buffer_rsrc_t r, int off, uint32_t* out) {
  if constexpr (W == 0) {
    out[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
  } else if constexpr (W == 1) {
    out[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
  } else if constexpr (W == 2) {
    const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
    out[0] = v[0], out[1] = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const u32x4 v = buffer_load16<false>(r, off + 16 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) out[4 * i + j] = v[j];
    }
  }
}
template <int W>
__device__ __forceinline__ void memory_words(const uint8_t* p, uint32_t* out) {
  if constexpr (W == 0) {
    out[0] = *(const uint16_t*)p;
  } else if constexpr (W == 1) {
    out[0] = *(const uint32_t*)p;
  } else if constexpr (W == 2) {
    const u32x2 v = ld8(p);
    out[0] = v[0], out[1] = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const u32x4 v = ld16(p + 16 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) out[4 * i + j] = v[j];
    }
  }
}

template <int D, class E, bool I4, bool PAGED, bool SCORES, int RT>
__global__ void __launch_bounds__(kCacheWaves * 64) attn_cache_kernel(const CacheArgs a) {
  static_assert(!PAGED || I4, "16-bit pools have kernels of their own");
  constexpr int ROW_BYTES = I4 ? D / 2 : 2 * D;
  constexpr int KS = D / 32;                      // k-steps of S^T
  constexpr int KW = ROW_BYTES / 16;              // words of a key row that a lane holds
  constexpr int VN = D / 16;                      // channels of a key that a lane holds, for V
  constexpr int VW = I4 ? VN / 8 : VN / 2;        // and their words (I4, D=64: 0, a half)
  constexpr int VR = VW == 0 ? 1 : VW;            // registers
  constexpr float NEG_INF = -__builtin_inff();
  using PV = typename std::conditional<I4, BF16, E>::type;  // element type of the second product

  __shared__ int table[PAGED ? kMaxSlots : 1];
  // (scale, zero) of a wave's tile as the products use them: K's 32 keys, then V's
  __shared__ __align__(16) float pairs[I4 ? kCacheWaves : 1][I4 ? 2 * kTile * 2 : 4];
  __shared__ __align__(16) float merge_o[2][16 * RT][D + 4];
  __shared__ float merge_ml[2][16 * RT][2];

  // ---- work item --------------------------------------------------------------------------------------------
  int rb, part, kvh, b;
  if (a.seqlens_k != nullptr) {
    // lengths differ: items are dealt to the XCDs one by one, partition outermost, so that those past a short
    // sequence's end come last (as in the paged split-K kernel); the row blocks of an item share an XCD's L2
    const int xcd = (int)blockIdx.x % 8, slot = (int)blockIdx.x / 8;
    rb = slot % a.n_rowblk;
    int item = (slot / a.n_rowblk) * 8 + xcd;
    if (item >= a.n_items) return;
    kvh = item % a.hkv;
    item /= a.hkv;
    b = item % a.batch;
    part = item / a.batch;
  } else {
    const int logical = xcd_remap((int)blockIdx.x, a.total);
    rb = logical % a.n_rowblk;
    int item = logical / a.n_rowblk;
    part = item % a.n_split;
    item /= a.n_split;
    kvh = item % a.hkv;
    b = item / a.hkv;
  }
  const int seq_q = a.nq;
  const int seq_k = a.seqlens_k != nullptr ? min(max(__builtin_amdgcn_readfirstlane(a.seqlens_k[b]), 0), a.nk) : a.nk;
  const int klo = part * a.split_len;
  // partitions past the sequence's end are not written, and not read by the combine
  if (a.seqlens_k != nullptr && klo >= seq_k) return;

  const int R = a.group * seq_q, r0 = rb * 16 * RT;
  const int tid = (int)threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // keys that any row, and that every row, of the block sees
  const int offset = seq_k - seq_q;  // bottom-right causal alignment
  int khi = min(seq_k, klo + a.split_len), mask_from;
  {
    const int re = min(r0 + 16 * RT, R);
    const bool wraps = re - r0 >= seq_q || (r0 % seq_q) > ((re - 1) % seq_q);
    const int qlo = wraps ? 0 : r0 % seq_q, qhi = wraps ? seq_q - 1 : (re - 1) % seq_q;
    if (a.causal) khi = min(khi, qhi + offset + 1);
    mask_from = a.causal ? min(khi, qlo + offset + 1) : khi;
  }
  const int n_tiles = khi > klo ? (khi - klo + kTile - 1) / kTile : 0;

  const int64_t krow = a.skn * (I4 ? 1 : 2), vrow = a.svn * (I4 ? 1 : 2);
  const uint8_t* kbase = (const uint8_t*)a.k + ((PAGED ? 0 : b * a.skb) + kvh * a.skh) * (I4 ? 1 : 2);
  const uint8_t* vbase = (const uint8_t*)a.v + ((PAGED ? 0 : b * a.svb) + kvh * a.svh) * (I4 ? 1 : 2);

  // paged: the partition's block-table entries; -1 where the page lies outside the pool
  int first_slot = 0;
  auto slot_of = [&](int n) __attribute__((always_inline)) {  // n / page_size
    return (int)(((uint64_t)(uint32_t)n * a.page_magic) >> a.page_magic_shift);
  };
  if constexpr (PAGED) {
    first_slot = slot_of(klo);
    const int slots = khi > klo ? slot_of(khi - 1) - first_slot + 1 : 0;  // <= 257 (host)
    for (int i = tid; i < slots; i += kCacheWaves * 64) {
      const int page = a.block_table[b * a.sbt + first_slot + i];
      table[i] = (uint32_t)page < (uint32_t)a.num_pages ? page : -1;
    }
    __syncthreads();
  }

  // ---- Q: B operands, and the sum of each row -------------------------------------------------------------
  u32x4 qf[RT][KS];
  float qsum[RT];
  int qlim[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = r0 + 16 * t + c;
    const bool ok = row < R;
    const int qh = ok ? row / seq_q : 0, qi = ok ? row % seq_q : 0;
    qlim[t] = qi + offset;
    const uint16_t* qp = (const uint16_t*)a.q + b * a.sqb + (kvh * a.group + qh) * a.sqh + qi * a.sqn;
    const uint32_t keep = ok ? 0xffffffffu : 0u;
    float s = 0.f;
#pragma unroll
    for (int m = 0; m < KS; ++m) {
      // 4 bits: word g * KS + m of a key row, whose operand pairs nibbles j and j + 4
      const int w = I4 ? g * KS + m : 4 * m + g;
      u32x4 v = ld16(qp + 8 * w) & keep;
      if constexpr (I4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s += lo_f32<E>(v[j]) + hi_f32<E>(v[j]);
        v = u32x4{pair_lo(v[0], v[2]), pair_hi(v[0], v[2]), pair_lo(v[1], v[3]), pair_hi(v[1], v[3])};
      }
      qf[t][m] = v;
    }
    qsum[t] = I4 ? sum_groups(s) : 0.f;
  }

  const float cs = a.qk_scale;  // of any sign, or 0: masked scores are set to -inf after it

  // ---- loads ------------------------------------------------------------------------------------------------
  // K block t, row c: key 8 (c / 4) + 4 t + c % 4 of the tile, words of channel group g.  V slot s: key 8 g + s.
  const int kkey = 8 * (c >> 2) + (c & 3);
  const int kpart = I4 ? g * KW * 4 : g * 16;  // bytes into the row (16 bit: + 64 a k-step)
  const int vpart = c * (VN * (I4 ? 1 : 4)) / 2;
  struct KTile {
    uint32_t w[2][KW];
  };
  struct VTile {
    uint32_t w[8][VR];
  };
  auto load_k_row = [&](auto&& get, uint32_t* w) __attribute__((always_inline)) {
    if constexpr (I4) {
      get(std::integral_constant<int, KW>{}, 0, w);
    } else {
#pragma unroll
      for (int m = 0; m < KS; ++m) get(std::integral_constant<int, 4>{}, 64 * m, w + 4 * m);
    }
  };
  // paged: a lane's rows of a tile lie in one page each for K and V (runs of 8 keys; pages are multiples of 16).
  // Keys past khi and pages outside the pool read page 0, which exists, and count as zero keys or are masked.
  auto page_row = [&](const uint8_t* base, int64_t spage, int64_t srow, int key) __attribute__((always_inline)) {
    const int slot = slot_of(key);
    const int page = key < khi ? table[slot - first_slot] : -1;
    const int64_t row = page >= 0 ? (int64_t)(key - slot * a.page_size) : 0;
    return base + max(page, 0) * spage + row * srow;
  };
  auto load_k = [&](int n0, KTile& t) __attribute__((always_inline)) {
    if constexpr (PAGED) {
      const uint8_t* p = page_row(kbase, a.skb, krow, n0 + 8 * (c >> 2)) + (c & 3) * krow + kpart;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        load_k_row([&](auto w, int off, uint32_t* out) { memory_words<decltype(w)::value>(p + 4 * u * krow + off, out); },
                   t.w[u]);
    } else {
      // a load past the limit returns zeros: rows at or past khi
      const int valid = min(khi - n0, kTile);
      const auto r = make_rsrc(kbase + n0 * krow, (uint32_t)(valid - 1) * (uint32_t)krow + ROW_BYTES);
#pragma unroll
      for (int u = 0; u < 2; ++u)
        load_k_row([&](auto w, int off, uint32_t* out) {
          buffer_words<decltype(w)::value>(r, (kkey + 4 * u) * (int)krow + kpart + off, out);
        }, t.w[u]);
    }
  };
  auto load_v = [&](int n0, VTile& t) __attribute__((always_inline)) {
    if constexpr (PAGED) {
      const uint8_t* p = page_row(vbase, a.svb, vrow, n0 + 8 * g) + vpart;
#pragma unroll
      for (int s = 0; s < 8; ++s) memory_words<VW>(p + s * vrow, t.w[s]);
    } else {
      const int valid = min(khi - n0, kTile);
      const auto r = make_rsrc(vbase + n0 * vrow, (uint32_t)(valid - 1) * (uint32_t)vrow + ROW_BYTES);
#pragma unroll
      for (int s = 0; s < 8; ++s) buffer_words<VW>(r, (8 * g + s) * (int)vrow + vpart, t.w[s]);
    }
  };
  // lane l: the pair of K (l < 32) or V of key l % 32 of the tile; zero past khi and outside the pool
  auto load_pair = [&](int n0) __attribute__((always_inline)) -> uint32_t {
    if constexpr (!I4) return 0u;
    const int key = n0 + (lane & 31);
    const bool kv = lane >= 32;
    const uint32_t* base = (const uint32_t*)(kv ? a.v_scale : a.k_scale) + kvh * (kv ? a.svsh : a.sksh);
    int64_t at = b, slot = key;
    bool ok = key < khi;
    if constexpr (PAGED) {
      const int sl = slot_of(key);
      at = ok ? table[sl - first_slot] : -1;
      ok = at >= 0;
      slot = key - sl * a.page_size;
    }
    uint32_t v = 0;
    if (ok) v = base[at * (kv ? a.svsb : a.sksb) + slot * (kv ? a.svsn : a.sksn)];
    return v;
  };

  f32x4 oacc[RT][VN];
  float m_run[RT], l_run[RT], psum[RT], zsum[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
#pragma unroll
    for (int n = 0; n < VN; ++n) oacc[t][n] = f32x4{};
    m_run[t] = NEG_INF;
    l_run[t] = psum[t] = zsum[t] = 0.f;
  }

  // ---- one tile: s (log2 domain), then p and O ---------------------------------------------------------------
  auto scores_of = [&](const KTile& kt, int n0, float(&s)[RT][8]) __attribute__((always_inline)) {
    f32x4 acc[RT][2];
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t][0] = acc[t][1] = f32x4{-qsum[t], -qsum[t], -qsum[t], -qsum[t]};
#pragma unroll
    for (int m = 0; m < KS; ++m) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        u32x4 ka;
        if constexpr (I4) {
          const uint32_t w = kt.w[u][m];
          ka = u32x4{codes2<E, 0>(w), codes2<E, 1>(w), codes2<E, 2>(w), codes2<E, 3>(w)};
        } else {
          ka = u32x4{kt.w[u][4 * m], kt.w[u][4 * m + 1], kt.w[u][4 * m + 2], kt.w[u][4 * m + 3]};
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[t][u] = mfma16<E>(ka, qf[t][m], acc[t][u]);
      }
    }
    if constexpr (I4) {
      const f32x4* kp = (const f32x4*)&pairs[wave][8 * g * 2];  // keys 8g..8g+7: (scale, zero) each
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 p = kp[i];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          s[t][2 * i] = __builtin_fmaf(acc[t][i >> 1][(2 * i) & 3], p[0], p[1] * qsum[t]);
          s[t][2 * i + 1] = __builtin_fmaf(acc[t][i >> 1][(2 * i + 1) & 3], p[2], p[3] * qsum[t]);
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
#pragma unroll
        for (int i = 0; i < 8; ++i) s[t][i] = acc[t][i >> 2][i & 3] * cs;
      }
    }
    if constexpr (SCORES) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int row = r0 + 16 * t + c;
        if (row < R) {
          float* out = a.raw + ((int64_t)(b * a.hkv + kvh) * R + row) * a.raw_stride + n0 + 8 * g;
          st16(out, __builtin_bit_cast(u32x4, f32x4{s[t][0], s[t][1], s[t][2], s[t][3]}));
          st16(out + 4, __builtin_bit_cast(u32x4, f32x4{s[t][4], s[t][5], s[t][6], s[t][7]}));
        }
      }
    }
    if (n0 + kTile > mask_from) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int end = a.causal ? min(khi, qlim[t] + 1) : khi;
#pragma unroll
        for (int i = 0; i < 8; ++i) s[t][i] = n0 + 8 * g + i < end ? s[t][i] : NEG_INF;
      }
    }
  };
  auto add_values = [&](const VTile& vt, float(&s)[RT][8]) __attribute__((always_inline)) {
    u32x4 pf[RT];
    f32x4 vp[4];
    if constexpr (I4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) vp[i] = ((const f32x4*)&pairs[wave][2 * kTile + 8 * g * 2])[i];
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float mt = s[t][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mt = vmax(mt, s[t][i]);
      const float m_new = vmax(m_run[t], max_groups(mt));
      // the maximum follows only when a row outgrows it by 2^8 (p <= 256 until then: O and l share it)
      if (__builtin_amdgcn_ballot_w64(m_new > m_run[t] + kRescaleLog2) != 0) {
        const float alpha = fast_exp2(m_run[t] - (m_new == NEG_INF ? 0.f : m_new));
        l_run[t] *= alpha, psum[t] *= alpha, zsum[t] *= alpha;
#pragma unroll
        for (int n = 0; n < VN; ++n) oacc[t][n] *= alpha;
        m_run[t] = m_new;
      }
      const float m = m_run[t] == NEG_INF ? 0.f : m_run[t];
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = fast_exp2(s[t][i] - m);
        l_run[t] += p[i];
      }
      if constexpr (I4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          zsum[t] = __builtin_fmaf(p[2 * i], vp[i][1], zsum[t]);
          zsum[t] = __builtin_fmaf(p[2 * i + 1], vp[i][3], zsum[t]);
          pf[t][i] = pack2<PV>(p[2 * i] * vp[i][0], p[2 * i + 1] * vp[i][2]);
          psum[t] = sum2<PV>(pf[t][i], psum[t]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) pf[t][i] = pack2<PV>(p[2 * i], p[2 * i + 1]);
      }
    }
    // A operands of channel n: its value for keys 8g .. 8g+7, two a register
    if constexpr (I4) {
#pragma unroll
      for (int h = 0; h < (VN + 3) / 4; ++h) {  // halves of 4 channels
        uint32_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t ka = vt.w[2 * j][h / 2], kb = vt.w[2 * j + 1][h / 2];
          x[j] = h & 1 ? pair_hi(ka, kb) : pair_lo(ka, kb);
        }
        const u32x4 v0 = {codes2<BF16, 0>(x[0]), codes2<BF16, 0>(x[1]), codes2<BF16, 0>(x[2]), codes2<BF16, 0>(x[3])};
        const u32x4 v1 = {codes2<BF16, 1>(x[0]), codes2<BF16, 1>(x[1]), codes2<BF16, 1>(x[2]), codes2<BF16, 1>(x[3])};
        const u32x4 v2 = {codes2<BF16, 2>(x[0]), codes2<BF16, 2>(x[1]), codes2<BF16, 2>(x[2]), codes2<BF16, 2>(x[3])};
        const u32x4 v3 = {codes2<BF16, 3>(x[0]), codes2<BF16, 3>(x[1]), codes2<BF16, 3>(x[2]), codes2<BF16, 3>(x[3])};
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          oacc[t][4 * h] = mfma16<PV>(v0, pf[t], oacc[t][4 * h]);
          oacc[t][4 * h + 1] = mfma16<PV>(v1, pf[t], oacc[t][4 * h + 1]);
          oacc[t][4 * h + 2] = mfma16<PV>(v2, pf[t], oacc[t][4 * h + 2]);
          oacc[t][4 * h + 3] = mfma16<PV>(v3, pf[t], oacc[t][4 * h + 3]);
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < VN / 2; ++h) {
        u32x4 lo, hi;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          lo[j] = pair_lo(vt.w[2 * j][h], vt.w[2 * j + 1][h]);
          hi[j] = pair_hi(vt.w[2 * j][h], vt.w[2 * j + 1][h]);
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          oacc[t][2 * h] = mfma16<PV>(lo, pf[t], oacc[t][2 * h]);
          oacc[t][2 * h + 1] = mfma16<PV>(hi, pf[t], oacc[t][2 * h + 1]);
        }
      }
    }
  };
  // the tile's pairs through LDS: each lane converts one, every lane reads eight keys'
  auto store_pair = [&](uint32_t w) __attribute__((always_inline)) {
    if constexpr (I4) {
      const float sc = lo_f32<F16>(w), z = hi_f32<F16>(w);
      const bool kv = lane >= 32;
      const f32x2 v = {16.f * sc * (kv ? 1.f : cs), kv ? __builtin_fmaf(7.5f, sc, z) : z * cs};
      *(f32x2*)&pairs[wave][2 * lane] = v;
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  };

  if (wave < n_tiles) {
    KTile kt;
    VTile vt;
    float s[RT][8];
    int n0 = klo + wave * kTile;
    load_k(n0, kt);
    uint32_t pr = load_pair(n0);
    load_v(n0, vt);
    for (int t = wave; t < n_tiles; t += kCacheWaves, n0 += kCacheWaves * kTile) {
      const bool more = t + kCacheWaves < n_tiles;
      const int next = n0 + kCacheWaves * kTile;
      if constexpr (I4) {
        // the next tile's words are few: all of them are in flight while this tile is worked on
        KTile kn;
        VTile vn;
        uint32_t pn = 0;
        store_pair(pr);
        if (more) {
          load_k(next, kn);
          pn = load_pair(next);
          load_v(next, vn);
        }
        scores_of(kt, n0, s);
        add_values(vt, s);
        kt = kn;
        vt = vn;
        pr = pn;
      } else {
        // K's registers are refilled once its product has read them, V's likewise
        scores_of(kt, n0, s);
        if (more) load_k(next, kt);
        add_values(vt, s);
        if (more) load_v(next, vt);
      }
    }
  }

  // ---- merge the waves, 2 and 3 into 0 and 1, then 1 into 0 ------------------------------------------------------
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    l_run[t] = sum_groups(l_run[t]);
    if constexpr (I4) {
      const float corr = sum_groups(zsum[t]) - (1.f + 7.5f / 16.f) * sum_groups(psum[t]);
#pragma unroll
      for (int n = 0; n < VN; ++n) oacc[t][n] += corr;
    }
  }
#pragma unroll
  for (int step = 2; step >= 1; step /= 2) {
    if (wave >= step && wave < 2 * step) {
      const int w = wave - step;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int row = 16 * t + c;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int n = 0; n < VN; n += 4)
            *(f32x4*)&merge_o[w][row][VN * (4 * g + i) + n] =
                f32x4{oacc[t][n][i], oacc[t][n + 1][i], oacc[t][n + 2][i], oacc[t][n + 3][i]};
        }
        if (g == 0) merge_ml[w][row][0] = m_run[t], merge_ml[w][row][1] = l_run[t];
      }
    }
    __syncthreads();
    if (wave < step) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int row = 16 * t + c;
        const float m2 = merge_ml[wave][row][0], l2 = merge_ml[wave][row][1];
        const float m = vmax(m_run[t], m2), ms = m == NEG_INF ? 0.f : m;
        const float f1 = fast_exp2(m_run[t] - ms), f2 = fast_exp2(m2 - ms);
        m_run[t] = m;
        l_run[t] = l_run[t] * f1 + l2 * f2;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int n = 0; n < VN; n += 4) {
            const f32x4 o2 = *(const f32x4*)&merge_o[wave][row][VN * (4 * g + i) + n];
#pragma unroll
            for (int j = 0; j < 4; ++j) oacc[t][n + j][i] = oacc[t][n + j][i] * f1 + o2[j] * f2;
          }
        }
      }
    }
    __syncthreads();
  }
  if (wave != 0) return;

  // ---- the partition's partial, normalised by its own sum, and (max, sum) -------------------------------------
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = r0 + 16 * t + c;
    if (row >= R) continue;
    const int hq = kvh * a.group + row / seq_q, qi = row % seq_q;
    const int64_t prow = ((int64_t)(b * a.hq + hq) * seq_q + qi) * a.n_split + part;
    const float inv = l_run[t] > 0.f ? 1.f / l_run[t] : 0.f;
    float* op = a.part + prow * D;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int n = 0; n < VN; n += 4)
        st16(op + VN * (4 * g + i) + n,
             __builtin_bit_cast(u32x4, f32x4{oacc[t][n][i] * inv, oacc[t][n + 1][i] * inv, oacc[t][n + 2][i] * inv,
                                             oacc[t][n + 3][i] * inv}));
    }
    if (g == 0) st8(a.ml + prow * 2, __builtin_bit_cast(u32x2, f32x2{m_run[t], l_run[t]}));
  }
}

// score_j = before_j + sum over the rows of 2^(s_rj - lse2_r), for the keys that a row sees.
// Four keys a thread; the rows' log-sum-exps are read through the scalar cache.
__global__ void __launch_bounds__(256) score_finish_kernel(const FinishArgs a) {
  const int bh = (int)(blockIdx.x / (uint32_t)a.chunks), b = bh / a.hkv, kvh = bh - b * a.hkv;
  const int seq_k = a.seqlens_k != nullptr ? min(max(a.seqlens_k[b], 0), a.nk) : a.nk;
  const int j = ((int)(blockIdx.x - (uint32_t)bh * (uint32_t)a.chunks) * 256 + (int)threadIdx.x) * 4;
  if (j >= a.nk) return;
  f32x4 w = {};
  if (j < seq_k) {
    const int R = a.group * a.nq, offset = seq_k - a.nq;
    const float* raw = a.raw + (int64_t)bh * R * a.raw_stride + j;
    for (int r = 0; r < R; ++r) {
      const int gi = r / a.nq, qi = r - gi * a.nq;
      const float lse = a.lse[b * a.slb + (kvh * a.group + gi) * a.slh + qi] * kLog2e;
      const int end = a.causal ? min(seq_k, qi + offset + 1) : seq_k;
      if (j >= end || lse == -__builtin_inff()) continue;  // (-inf: every key of the row scores -inf)
      const f32x4 s = __builtin_bit_cast(f32x4, ld16(raw + r * a.raw_stride));
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] += j + i < end ? fast_exp2(s[i] - lse) : 0.f;
    }
  }
  const float* in = a.in != nullptr ? a.in + b * a.sib + kvh * a.sih : nullptr;
  float* out = a.out + b * a.sob + kvh * a.soh;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (j + i < a.nk) out[j + i] = w[i] + (in != nullptr ? in[j + i] : 0.f);
  }
}

template <int D, class E, bool I4, bool PAGED, bool SCORES>
hipError_t launch_rows(const CacheArgs& a, int rt, hipStream_t stream) {
  if (rt == 1) {
    hipLaunchKernelGGL((attn_cache_kernel<D, E, I4, PAGED, SCORES, 1>), dim3((unsigned)a.total), dim3(kCacheWaves * 64),
                       0, stream, a);
  } else {
    hipLaunchKernelGGL((attn_cache_kernel<D, E, I4, PAGED, SCORES, 2>), dim3((unsigned)a.total), dim3(kCacheWaves * 64),
                       0, stream, a);
  }
  return hipGetLastError();
}

template <int D, class E>
hipError_t launch_cache(const CacheArgs& a, bool i4, bool paged, bool scores, int rt, hipStream_t stream) {
  if (!i4) return launch_rows<D, E, false, false, true>(a, rt, stream);
  if (paged) return launch_rows<D, E, true, true, false>(a, rt, stream);
  return scores ? launch_rows<D, E, true, false, true>(a, rt, stream)
                : launch_rows<D, E, true, false, false>(a, rt, stream);
}

int64_t raw_stride(const fa_cache_params& p) { return ((int64_t)p.seqlen_k + kTile - 1) / kTile * kTile; }

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

int splits(const fa_cache_params& p, int split_len) {
  return p.seqlen_k > 0 ? (p.seqlen_k + split_len - 1) / split_len : 1;
}

}  // namespace

size_t cache_workspace_bytes(const fa_cache_params& p, int32_t split_len) {
  size_t need = align16(fa_splitk_workspace_bytes(p.batch, p.heads_q, p.seqlen_q, p.head_dim, splits(p, split_len)));
  if (p.scores_out != nullptr) {
    const size_t rows = (size_t)p.batch * p.heads_q * p.seqlen_q;
    need += align16(rows * sizeof(float)) + rows * (size_t)raw_stride(p) * sizeof(float);
  }
  return need;
}

fa_status run_cache(const fa_cache_params& p, int32_t split_len, void* workspace, hipStream_t stream, const char** err) {
  CacheArgs a{};
  const int S = splits(p, split_len);
  const bool i4 = p.kv_dtype == FA_DTYPE_INT4, paged = p.block_table != nullptr, scores = p.scores_out != nullptr;
  a.q = p.q, a.k = p.k, a.v = p.v, a.k_scale = p.k_scale, a.v_scale = p.v_scale;
  a.sqb = p.q_stride_b, a.sqh = p.q_stride_h, a.sqn = p.q_stride_n;
  a.skb = p.k_stride_b, a.skh = p.k_stride_h, a.skn = p.k_stride_n;
  a.svb = p.v_stride_b, a.svh = p.v_stride_h, a.svn = p.v_stride_n;
  a.sksb = p.k_scale_stride_b, a.sksh = p.k_scale_stride_h, a.sksn = p.k_scale_stride_n;
  a.svsb = p.v_scale_stride_b, a.svsh = p.v_scale_stride_h, a.svsn = p.v_scale_stride_n;
  a.batch = p.batch, a.hq = p.heads_q, a.hkv = p.heads_kv, a.group = p.heads_q / p.heads_kv;
  a.nq = p.seqlen_q, a.nk = p.seqlen_k;
  a.qk_scale = p.scale * kLog2e;
  a.causal = p.causal ? 1 : 0;
  a.n_split = S, a.split_len = split_len;
  a.seqlens_k = p.seqlens_k;
  a.block_table = p.block_table, a.sbt = p.block_table_stride, a.num_pages = p.num_pages, a.page_size = p.page_size;
  if (paged) {
    int lg = 0;
    while ((int64_t{1} << lg) < (int64_t)p.page_size) ++lg;
    a.page_magic_shift = 31 + lg;
    a.page_magic = (uint32_t)(((uint64_t{1} << a.page_magic_shift) + (uint64_t)p.page_size - 1) / (uint64_t)p.page_size);
    if (((int64_t)split_len - 1) / p.page_size + 2 > kMaxSlots) {
      *err = "split_len too long for the page size: a partition may span at most 258 pages";
      return FA_ERR_UNSUPPORTED;
    }
  }
  const int rows = a.group * p.seqlen_q, rt = rows <= 16 ? 1 : 2;
  a.n_rowblk = (rows + 16 * rt - 1) / (16 * rt);
  const int64_t items = (int64_t)p.batch * p.heads_kv * S, out_rows = (int64_t)p.batch * p.heads_q * p.seqlen_q;
  const int64_t total = (p.seqlens_k != nullptr ? (items + 7) / 8 * 8 : items) * a.n_rowblk;
  if (total > INT32_MAX || out_rows > INT32_MAX) {
    *err = "grid too large";
    return FA_ERR_UNSUPPORTED;
  }
  a.total = (int32_t)total;
  a.n_items = (int32_t)items;
  uint8_t* ws = (uint8_t*)workspace;
  a.part = (float*)ws;
  a.ml = a.part + out_rows * S * p.head_dim;
  float* lse = p.lse;
  int64_t slb = p.lse_stride_b, slh = p.lse_stride_h;
  if (scores) {
    float* own = (float*)(ws + align16(fa_splitk_workspace_bytes(p.batch, p.heads_q, p.seqlen_q, p.head_dim, S)));
    a.raw = (float*)((uint8_t*)own + align16((size_t)out_rows * sizeof(float)));
    a.raw_stride = raw_stride(p);
    if (lse == nullptr) lse = own, slb = (int64_t)p.heads_q * p.seqlen_q, slh = p.seqlen_q;
  }
  const bool bf = p.dtype == FA_DTYPE_BF16;
  hipError_t e = hipErrorInvalidValue;
  if (p.head_dim == 64) {
    e = bf ? launch_cache<64, BF16>(a, i4, paged, scores, rt, stream) : launch_cache<64, F16>(a, i4, paged, scores, rt, stream);
  } else if (p.head_dim == 128) {
    e = bf ? launch_cache<128, BF16>(a, i4, paged, scores, rt, stream) : launch_cache<128, F16>(a, i4, paged, scores, rt, stream);
  } else if (p.head_dim == 256) {
    e = bf ? launch_cache<256, BF16>(a, i4, paged, scores, rt, stream) : launch_cache<256, F16>(a, i4, paged, scores, rt, stream);
  }
  if (e != hipSuccess) return hip_status(e, err);

  CombineArgs c{};
  c.opart = a.part, c.ml = a.ml, c.o = p.o;
  c.sob = p.o_stride_b, c.soh = p.o_stride_h, c.son = p.o_stride_n;
  c.lse = lse, c.slb = slb, c.slh = slh;
  c.hq = p.heads_q, c.group = a.group, c.nq = p.seqlen_q, c.n_split = S;
  c.seqlens_k = p.seqlens_k, c.nk = p.seqlen_k, c.split_len = split_len;
  const fa_status st = run_combine(c, p.head_dim, bf, out_rows, stream, err);
  if (st != FA_OK || !scores) return st;

  FinishArgs f{};
  f.raw = a.raw, f.raw_stride = a.raw_stride;
  f.lse = lse, f.slb = slb, f.slh = slh;
  f.in = p.scores_in, f.sib = p.scores_in_stride_b, f.sih = p.scores_in_stride_h;
  f.out = p.scores_out, f.sob = p.scores_out_stride_b, f.soh = p.scores_out_stride_h;
  f.seqlens_k = p.seqlens_k;
  f.hkv = p.heads_kv, f.group = a.group, f.nq = p.seqlen_q, f.nk = p.seqlen_k, f.causal = a.causal;
  if (p.seqlen_k == 0) return FA_OK;
  f.chunks = (p.seqlen_k - 1) / 1024 + 1;
  const int64_t blocks = (int64_t)p.batch * p.heads_kv * f.chunks;
  if (blocks > INT32_MAX) {
    *err = "grid too large";
    return FA_ERR_UNSUPPORTED;
  }
  hipLaunchKernelGGL(score_finish_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, f);
  return hip_status(hipGetLastError(), err);
}

}  // namespace fa
