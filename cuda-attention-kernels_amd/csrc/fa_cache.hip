// Attention over a 4-bit K/V cache, and attention that scores the keys of its cache (4-bit or 16-bit).
//
// For queries q_r (the G * n_q (q-head, query) rows that share a kv-head) and keys j of the first seqlens_k[b]:
//   K_j = ks_j kc_j + kz_j,  V_j = vs_j vc_j + vz_j        (kc, vc: D codes of 4 bits; one fp16 pair a row)
//   s_rj = c q_r . K_j,  p_rj = 2^(s_rj - m_r),  o_r = sum_j p_rj V_j / sum_j p_rj     (c = scale * log2 e)
//   score_j = sum_r p_rj / sum_j' p_rj'                                               (attention_scored)
//
// Decomposition.  Keys are cut into partitions of split_len; a workgroup of four waves takes one partition of one
// (batch, kv-head) for up to 16 * RT rows, its waves every fourth 32-key tile each (scored calls of up to 16 rows: a run
// of tiles each, whose scores are written together); the waves' (m, l, O) are merged through LDS into one fp32 partial,
// and cache_finish_kernel or splitk_combine_kernel merges the partitions.  Bound by
// the bytes of the cache (D + 8 a key at 4 bits, 4 D at 16) up to 16 rows of D=128: bf16, 32 x 8 heads x 32768 keys
// (1.14 GB) 177 us = 6.4 TB/s.  Bound by the vector unit beyond that (codes, exponentials: 8 x 8 heads x 64 rows of
// D=256, 20000 keys, 342 MB and 84 GFLOP: 146 us) and at D=64, where a key's few bytes need the same exponentials (48 x
// 8 heads of ragged lengths to 8000, 103 MB: 47 us).
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
// so that P's rounding (2^-8 of itself) meets only (code - 7.5)/16, at most 0.47 of it.  For fp16 outputs, whose own
// rounding is 2^-11, P' is the sum of two bf16 terms and takes two products.  Everything else is fp32.
//
// Scores.  p needs the row's final sum, which no partition has.  The s of a row and key are written as they are, and
// cache_finish_kernel reads them and turns them into weights once the partitions' sums are there: 8 bytes for every row of
// a key, in all.  A second pass over K would read 2 D bytes of a key instead (4 bits: D/2 + 4), so this moves less up to
// about D/4 rows (D/16), 32 and 8 at D=128; the 128 rows of 8 heads x 8191 keys write 42 MB and read them again beside 34 MB
// of keys and values.  They lie tile by tile, the rows of 32 keys together, so that a workgroup writes one run of memory.
#include <algorithm>

#include "fa_device.hpp"
#include "fa_internal.hpp"

namespace fa {

namespace {

constexpr int kCacheWaves = 4;
constexpr int kTile = 32;         // keys a wave step
constexpr int kMaxSlots = 258;    // block-table entries of a partition (paged)
constexpr int kStageFloats = 2048;  // scores that a wave holds back

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

// Nibble n (0..3) of both halves of a word as two 16-bit floats 1 + code/16: a shift to the top of the mantissa and
// one v_and_or.  That takes one scalar operand and no literal, so the mask is kept in a vector register.
template <class E>
struct Codes {
  static constexpr int at = std::is_same<E, BF16>::value ? 3 : 6;
  uint32_t mask, one;
  __device__ __forceinline__ Codes() {
    mask = (0xfu << at) * 0x10001u;
    one = std::is_same<E, BF16>::value ? 0x3f803f80u : 0x3c003c00u;
    __asm__("" : "+v"(mask));
    __asm__("" : "+s"(one));
  }
  template <int N>
  __device__ __forceinline__ uint32_t get(uint32_t x) const {
    constexpr int sh = 4 * N - at;
    const uint32_t y = sh >= 0 ? x >> (sh & 31) : x << ((-sh) & 31);
    return (y & mask) | one;
  }
};

// halves {a.lo, b.lo} and {a.hi, b.hi}
__device__ __forceinline__ uint32_t pair_lo(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t pair_hi(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// W words (W = 0: one 16-bit half) of a buffer (AUX: its cache policy), or of memory
template <int W, int AUX>
__device__ __forceinline__ void buffer_words(__amdgpu_buffer_rsrc_t r, int off, uint32_t* out) {
  if constexpr (W == 0) {
    out[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, off, 0, AUX);
  } else if constexpr (W == 1) {
    out[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, AUX);
  } else if constexpr (W == 2) {
    const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, AUX));
    out[0] = v[0], out[1] = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const u32x4 v = buffer_load16<AUX != 0>(r, off + 16 * i);
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

// Waves a SIMD, which bound the registers: as many as fit without spilling, but for the cases named.  One row block of 4
// bits and D <= 128, or 16 bits and D = 64, holds three (4 bits, 32 x 8 heads x 32768 keys: 177 us, with two 188); 16 bits
// at D = 128 two (16 x 8 heads x 4 rows, 16384 keys: 208 us, with three and 6 registers spilled 219); more rows hold O in
// more registers.  D = 256 with 32 rows of 4 bits spills 30 to 47 registers at two waves, and is faster so than with one
// (148 and 178 us); 64 scored rows of D = 64 and fp16 spill 5 at two.
template <int D, bool I4, int RT>
constexpr int waves_per_simd() {
  if (RT == 4) return I4 && D == 64 ? 2 : 1;
  if (RT == 2) return D == 256 && !I4 ? 1 : 2;
  return D == 256 ? 1 : I4 || D == 64 ? 3 : 2;
}

template <int D, class E, bool I4, bool PAGED, bool SCORES, int RT>
__global__ void __launch_bounds__(kCacheWaves * 64) __attribute__((amdgpu_waves_per_eu(waves_per_simd<D, I4, RT>())))
attn_cache_kernel(const CacheArgs a) {
  static_assert(!PAGED || I4, "16-bit pools have kernels of their own");
  constexpr int ROW_BYTES = I4 ? D / 2 : 2 * D;
  constexpr int KS = D / 32;                      // k-steps of S^T
  constexpr int KW = ROW_BYTES / 16;              // words of a key row that a lane holds
  constexpr int VN = D / 16;                      // channels of a key that a lane holds, for V
  constexpr int VW = I4 ? VN / 8 : VN / 2;        // and their words (I4, D=64: 0, a half)
  constexpr int VR = VW == 0 ? 1 : VW;            // registers
  // Q's operands in LDS where two waves then fit a SIMD (8 x 8 heads x 64 rows, 20000 keys: D=256 178 us with one wave,
  // 146 so; D=64 77 and 75; at D=128 64 rows spill: 67 and 79)
  constexpr bool QLDS = I4 && ((RT == 4 && D == 64) || (D == 256 && RT == 2));
  // A cache row that one row block reads is read once: non-temporal (32 x 8 heads x 32768 keys: 183 us, cached 203).
  // Where several row blocks share it, the later ones find it in L2 (8 heads x 128 rows, 8191 keys: 24 us cached, 29 not).
  constexpr int AUX = RT == 1 ? 2 : 0;
  constexpr float NEG_INF = -__builtin_inff();
  using PV = typename std::conditional<I4, BF16, E>::type;  // element type of the second product
  // 4 bits, bf16: Q is taken 2^10 smaller (exact down to 2^-116) and the scores' multiplier larger, so that sum(q) and the
  // sums of q (1 + code/16) stay finite for every finite q
  constexpr float QDOWN = I4 && std::is_same<E, BF16>::value ? 1.f / 1024.f : 1.f;
  constexpr bool LOW = I4 && std::is_same<E, F16>::value;   // P as two bf16 terms: fp16 outputs keep their precision

  __shared__ int table[PAGED ? kMaxSlots : 1];
  // (scale, zero) of a wave's tile as the products use them: K's 32 keys, then V's
  __shared__ __align__(16) float pairs[I4 ? kCacheWaves : 1][I4 ? 2 * kTile * 2 : 4];
  // scored, up to 16 rows: the scores of a wave's last tiles, written out together
  constexpr bool STAGED = SCORES && RT == 1;
  __shared__ __align__(16) float stage[STAGED ? kCacheWaves : 1][STAGED ? kStageFloats : 4];
  __shared__ __align__(16) float merge_o[2][16 * RT][D + 4];
  __shared__ float merge_ml[2][16 * RT][2];
  u32x4(*const qlds)[64] = (u32x4(*)[64])merge_o;  // until the merge

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
  const int seq_q = a.nq, klo = part * a.split_len;
  const int tid = (int)threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // paged: the partition's block-table entries; -1 where the page lies outside the pool.  Bounded by the grid's largest
  // length, so that they do not wait for this sequence's.
  int first_slot = 0;
  auto slot_of = [&](int n) __attribute__((always_inline)) {  // n / page_size
    return (int)(((uint64_t)(uint32_t)n * a.page_magic) >> a.page_magic_shift);
  };
  if constexpr (PAGED) {
    first_slot = slot_of(klo);
    const int end = min(a.nk, klo + a.split_len);
    const int slots = end > klo ? slot_of(end - 1) - first_slot + 1 : 0;  // <= kMaxSlots (host)
    for (int i = tid; i < slots; i += kCacheWaves * 64) {
      const int page = a.block_table[b * a.sbt + first_slot + i];
      table[i] = (uint32_t)page < (uint32_t)a.num_pages ? page : -1;
    }
    __syncthreads();
  }
  const int seq_k = a.seqlens_k != nullptr ? min(max(__builtin_amdgcn_readfirstlane(a.seqlens_k[b]), 0), a.nk) : a.nk;
  // partitions past the sequence's end are not written, and not read by the combine
  if (a.seqlens_k != nullptr && klo >= seq_k) return;

  const int R = a.group * seq_q, r0 = rb * 16 * RT;

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

  const float cs = a.qk_scale / QDOWN;  // of any sign, or 0: masked scores are set to -inf after it

  // ---- loads ------------------------------------------------------------------------------------------------
  // K block u, row c: key 8 (c / 4) + 4 u + c % 4 of the tile, words of channel group g.  V slot i: key 8 g + i.
  struct Tile {
    uint32_t k[2][KW], v[8][VR], pair;
  };
  const int kkey = 8 * (c >> 2) + (c & 3);
  const int kpart = I4 ? g * KW * 4 : g * 16;  // bytes into the row (16 bit: + 64 a k-step)
  const int vpart = c * (VN * (I4 ? 1 : 4)) / 2;
  // rows that follow each other directly: the loads of a lane differ by constants, which the instructions hold
  const bool packed = krow == ROW_BYTES && vrow == ROW_BYTES;
  auto load_k_row = [&](auto&& get, uint32_t* w) __attribute__((always_inline)) {
    if constexpr (I4) {
      get(std::integral_constant<int, KW>{}, 0, w);
    } else {
#pragma unroll
      for (int m = 0; m < KS; ++m) get(std::integral_constant<int, 4>{}, 64 * m, w + 4 * m);
    }
  };
  // Dense: a descriptor a tile; a load past its limit returns zeros (rows at or past khi).
  auto load_k_dense = [&](int n0, Tile& t) __attribute__((always_inline)) {
    const int valid = min(khi - n0, kTile);
    const auto r = make_rsrc(kbase + n0 * krow, (uint32_t)(valid - 1) * (uint32_t)krow + ROW_BYTES);
    auto rows = [&](int row) __attribute__((always_inline)) {
      const int at = kkey * row + kpart;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        load_k_row([&](auto w, int off, uint32_t* out) { buffer_words<decltype(w)::value, AUX>(r, at + 4 * u * row + off, out); },
                   t.k[u]);
    };
    if (packed) rows(ROW_BYTES); else rows((int)krow);
  };
  auto load_v_dense = [&](int n0, Tile& t) __attribute__((always_inline)) {
    const int valid = min(khi - n0, kTile);
    const auto r = make_rsrc(vbase + n0 * vrow, (uint32_t)(valid - 1) * (uint32_t)vrow + ROW_BYTES);
    auto rows = [&](int row) __attribute__((always_inline)) {
      const int at = 8 * g * row + vpart;
#pragma unroll
      for (int i = 0; i < 8; ++i) buffer_words<VW, AUX>(r, at + i * row, t.v[i]);
    };
    if (packed) rows(ROW_BYTES); else rows((int)vrow);
  };
  // (scale, zero) words: lane l holds K's (l < 32) or V's of key l % 32 of the tile, zero past khi
  const bool vlane = lane >= kTile;
  const int64_t pstep = (vlane ? a.svsn : a.sksn) * 4;
  const uint8_t* pbase = (const uint8_t*)(vlane ? a.v_scale : a.k_scale) + kvh * (vlane ? a.svsh : a.sksh) * 4;
  if constexpr (I4 && !PAGED) pbase += b * (vlane ? a.svsb : a.sksb) * 4 + (int64_t)(lane & 31) * pstep;
  auto load_pair_dense = [&](int n0, Tile& t) __attribute__((always_inline)) {
    if constexpr (I4) {
      t.pair = 0;
      if (n0 + (lane & 31) < khi) t.pair = *(const uint32_t*)(pbase + n0 * pstep);
    }
  };
  // Paged: page sizes are multiples of 16, so each half of a tile lies in one page: a scalar base each, of which a lane
  // takes the one of its keys.  Halves past khi and pages outside the pool read page 0, which exists; their pairs are
  // zero (zero keys, or masked ones).
  auto load_paged = [&](int n0, Tile& t, auto do_k, auto do_v) __attribute__((always_inline)) {
    const uint8_t *kp[2], *vp[2];
    int64_t at[2];
    int off[2];
    bool ok[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = n0 + 16 * h, slot = slot_of(key);
      const int page = key < khi ? __builtin_amdgcn_readfirstlane(table[slot - first_slot]) : -1;
      ok[h] = page >= 0;
      at[h] = max(page, 0);
      off[h] = ok[h] ? key - slot * a.page_size : 0;
      kp[h] = kbase + at[h] * a.skb + off[h] * krow;
      vp[h] = vbase + at[h] * a.svb + off[h] * vrow;
    }
    const uint8_t* k = (c >= 8 ? kp[1] : kp[0]) + (kkey & 15) * (int)krow + kpart;
    const uint8_t* v = (g >= 2 ? vp[1] : vp[0]) + 8 * (g & 1) * (int)vrow + vpart;
    auto rows = [&](int kr, int vr) __attribute__((always_inline)) {
      if constexpr (do_k) {
#pragma unroll
        for (int u = 0; u < 2; ++u) memory_words<KW>(k + 4 * u * kr, t.k[u]);
      }
      if constexpr (do_v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) memory_words<VW>(v + i * vr, t.v[i]);
      }
    };
    if (packed) rows(ROW_BYTES, ROW_BYTES); else rows((int)krow, (int)vrow);
    if constexpr (!do_k) return;
    const int h = (lane >> 4) & 1;
    t.pair = 0;
    if ((h ? ok[1] : ok[0]) && n0 + (lane & 31) < khi) {
      const int64_t word = (h ? at[1] : at[0]) * (vlane ? a.svsb : a.sksb) * 4 + ((h ? off[1] : off[0]) + (lane & 15)) * pstep;
      t.pair = *(const uint32_t*)(pbase + word);
    }
  };
  using Yes = std::true_type;
  using No = std::false_type;
  auto load_k = [&](int n0, Tile& t) __attribute__((always_inline)) {  // and the pairs
    if constexpr (PAGED) {
      load_paged(n0, t, Yes{}, No{});
    } else {
      load_k_dense(n0, t);
      load_pair_dense(n0, t);
    }
  };
  auto load_v = [&](int n0, Tile& t) __attribute__((always_inline)) {
    if constexpr (PAGED) {
      load_paged(n0, t, No{}, Yes{});
    } else {
      load_v_dense(n0, t);
    }
  };
  auto load_tile = [&](int n0, Tile& t) __attribute__((always_inline)) {
    if constexpr (PAGED) {
      load_paged(n0, t, Yes{}, Yes{});
    } else {
      load_k(n0, t);
      load_v(n0, t);
    }
  };

  // the first tiles are on their way before anything waits for Q
  // (staged scores: a wave's tiles follow each other, else the waves take every fourth)
  constexpr int STEP = STAGED ? kTile : kCacheWaves * kTile;
  const int share = (n_tiles + kCacheWaves - 1) / kCacheWaves;
  int n0 = klo + (STAGED ? wave * share : wave) * kTile;
  const int last = klo + ((STAGED ? min((wave + 1) * share, n_tiles) : n_tiles) - 1) * kTile;  // the last tile's first key
  constexpr bool REFILL = !I4 || QLDS;  // one tile's registers, refilled as they are read
  Tile tiles[REFILL ? 1 : 2];
  if (n0 <= last) load_tile(n0, tiles[0]);

  // ---- Q: B operands, and the sum of each row -------------------------------------------------------------
  u32x4 qf[QLDS ? 1 : RT][QLDS ? 1 : KS];
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
        if constexpr (QDOWN != 1.f) {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = pack2<E>(lo_f32<E>(v[j]) * QDOWN, hi_f32<E>(v[j]) * QDOWN);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) s += lo_f32<E>(v[j]) + hi_f32<E>(v[j]);
        v = u32x4{pair_lo(v[0], v[2]), pair_hi(v[0], v[2]), pair_lo(v[1], v[3]), pair_hi(v[1], v[3])};
      }
      if constexpr (QLDS) {
        if (m % kCacheWaves == wave) qlds[t * KS + m][lane] = v;  // every wave holds the same
      } else {
        qf[t][m] = v;
      }
    }
    qsum[t] = I4 ? sum_groups(s) : 0.f;
  }
  if constexpr (QLDS) __syncthreads();

  f32x4 oacc[RT][VN];
  float m_run[RT], l_run[RT], psum[RT], zsum[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
#pragma unroll
    for (int n = 0; n < VN; ++n) oacc[t][n] = f32x4{};
    m_run[t] = NEG_INF;
    l_run[t] = psum[t] = zsum[t] = 0.f;
  }

  // ---- one tile -----------------------------------------------------------------------------------------------
  const Codes<E> kcodes;
  const Codes<BF16> vcodes;
  // S^T = K Q^T (4 bits: from -sum(q), so that it is q . code / 16)
  auto product_k = [&](const Tile& kt, f32x4(&acc)[RT][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t][0] = acc[t][1] = f32x4{-qsum[t], -qsum[t], -qsum[t], -qsum[t]};
#pragma unroll
    for (int m = 0; m < KS; ++m) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        u32x4 ka;
        if constexpr (I4) {
          const uint32_t w = kt.k[u][m];
          ka = u32x4{kcodes.template get<0>(w), kcodes.template get<1>(w), kcodes.template get<2>(w),
                     kcodes.template get<3>(w)};
        } else {
          ka = u32x4{kt.k[u][4 * m], kt.k[u][4 * m + 1], kt.k[u][4 * m + 2], kt.k[u][4 * m + 3]};
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          if constexpr (QLDS) {
            acc[t][u] = mfma16<E>(ka, qlds[t * KS + m][lane], acc[t][u]);
          } else {
            acc[t][u] = mfma16<E>(ka, qf[t][m], acc[t][u]);
          }
        }
      }
    }
  };
  // p = 2^(s - m), and O += P V
  float raw[SCORES ? RT : 1][8];  // scored: this tile's scores
  auto product_v = [&](const Tile& vt, f32x4(&acc)[RT][2], int n0) __attribute__((always_inline)) {
    u32x4 pf[RT], pl[RT];
    f32x4 kp[4], vp[4];
    if constexpr (I4) {  // keys 8g .. 8g+7: (multiplier of the product, multiplier of sum(q))
#pragma unroll
      for (int i = 0; i < 4; ++i) kp[i] = ((const f32x4*)&pairs[wave][8 * g * 2])[i];
    }
    float p[RT][8];
    const bool masked = n0 + kTile > mask_from;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int end = a.causal ? min(khi, qlim[t] + 1) : khi;
      // the scores less `m` (log2 domain)
      auto scores_less = [&](float m, float(&s)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = acc[t][i >> 2][i & 3];
          if constexpr (I4) {
            s[i] = __builtin_fmaf(x, kp[i >> 1][2 * (i & 1)], __builtin_fmaf(kp[i >> 1][2 * (i & 1) + 1], qsum[t], -m));
          } else {
            s[i] = __builtin_fmaf(x, cs, -m);
          }
        }
      };
      auto mask = [&](float(&s)[8]) __attribute__((always_inline)) {
        if (masked) {
#pragma unroll
          for (int i = 0; i < 8; ++i) s[i] = n0 + 8 * g + i < end ? s[i] : NEG_INF;
        }
      };
      float s[8];
      if constexpr (SCORES) {
        scores_less(0.f, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          raw[t][i] = s[i];
          s[i] -= m_run[t];
        }
      } else {
        scores_less(m_run[t], s);
      }
      mask(s);
      // The maximum follows only when a row outgrows it by 2^8 (p <= 256 until then: O and l share it): most tiles need
      // no exchange between the lanes of a row.  The first tile's m is -inf, and s then +inf (or NaN, of a score -inf).
      float mt = s[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mt = vmax(mt, s[i]);
      if (__builtin_amdgcn_ballot_w64(!(mt <= kRescaleLog2)) != 0) {
        scores_less(0.f, s);
        mask(s);
        mt = s[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mt = vmax(mt, s[i]);
        const float m_new = vmax(m_run[t], max_groups(mt)), m = m_new == NEG_INF ? 0.f : m_new;
        const float alpha = fast_exp2(m_run[t] - m);
        l_run[t] *= alpha, psum[t] *= alpha, zsum[t] *= alpha;
#pragma unroll
        for (int n = 0; n < VN; ++n) oacc[t][n] *= alpha;
        m_run[t] = m_new;
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] -= m;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[t][i] = fast_exp2(s[i]);
        l_run[t] += p[t][i];
      }
    }
    if constexpr (I4) {  // V's: 16 scale, and zero + 7.5 scale
#pragma unroll
      for (int i = 0; i < 4; ++i) vp[i] = ((const f32x4*)&pairs[wave][2 * kTile + 8 * g * 2])[i];
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (I4) {
          zsum[t] = __builtin_fmaf(p[t][2 * i], vp[i][1], zsum[t]);
          zsum[t] = __builtin_fmaf(p[t][2 * i + 1], vp[i][3], zsum[t]);
          const float x = p[t][2 * i] * vp[i][0], y = p[t][2 * i + 1] * vp[i][2];
          pf[t][i] = pack2<BF16>(x, y);
          psum[t] = sum2<BF16>(pf[t][i], psum[t]);
          if constexpr (LOW) {
            pl[t][i] = pack2<BF16>(x - lo_f32<BF16>(pf[t][i]), y - hi_f32<BF16>(pf[t][i]));
            psum[t] = sum2<BF16>(pl[t][i], psum[t]);
          }
        } else {
          pf[t][i] = pack2<E>(p[t][2 * i], p[t][2 * i + 1]);
        }
      }
    }
    // A operands of channel n: its value for keys 8g .. 8g+7, two a register
    auto channel = [&](int n, const u32x4& v) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        oacc[t][n] = mfma16<PV>(v, pf[t], oacc[t][n]);
        if constexpr (LOW) oacc[t][n] = mfma16<PV>(v, pl[t], oacc[t][n]);
      }
    };
    if constexpr (I4) {
#pragma unroll
      for (int h = 0; h < VN / 4; ++h) {  // halves of 4 channels
        uint32_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t ka = vt.v[2 * j][h / 2], kb = vt.v[2 * j + 1][h / 2];
          x[j] = h & 1 ? pair_hi(ka, kb) : pair_lo(ka, kb);
        }
        auto nibble = [&](auto n) __attribute__((always_inline)) {
          constexpr int N = decltype(n)::value;
          channel(4 * h + N, u32x4{vcodes.template get<N>(x[0]), vcodes.template get<N>(x[1]), vcodes.template get<N>(x[2]),
                                   vcodes.template get<N>(x[3])});
        };
        nibble(std::integral_constant<int, 0>{});
        nibble(std::integral_constant<int, 1>{});
        nibble(std::integral_constant<int, 2>{});
        nibble(std::integral_constant<int, 3>{});
      }
    } else {
#pragma unroll
      for (int h = 0; h < VN / 2; ++h) {
        u32x4 lo, hi;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          lo[j] = pair_lo(vt.v[2 * j][h], vt.v[2 * j + 1][h]);
          hi[j] = pair_hi(vt.v[2 * j][h], vt.v[2 * j + 1][h]);
        }
        channel(2 * h, lo);
        channel(2 * h + 1, hi);
      }
    }
  };
  // Staged: 33 MB of scores beside 1 GB of keys cost 60 us when every tile wrote its 512 bytes, 50 so, of 219 in all (what
  // is left is the memory's turning between reads and writes: writes that stay in the L2 cost 10; three waves a SIMD).
  // Direct: rows past R are beyond the descriptor's limit and dropped, without a branch around the stores (loads and
  // stores share one counter: a wait after stores that may have been skipped waits for too much).
  const int stage_tiles = STAGED ? kStageFloats / (R * kTile) : 1;
  int staged = 0;
  auto flush_scores = [&](int n0) __attribute__((always_inline)) {  // n0: the last staged tile
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float* out = a.raw + ((int64_t)(b * a.hkv + kvh) * a.raw_tiles + n0 / kTile - (staged - 1)) * R * kTile;
    for (int i = 4 * lane; i < staged * R * kTile; i += 256) st16(out + i, ld16(&stage[STAGED ? wave : 0][i]));
    __builtin_amdgcn_wave_barrier();
    staged = 0;
  };
  auto store_scores = [&](int n0) __attribute__((always_inline)) {
    if constexpr (STAGED) {
      if (c < R) {
        float* at = &stage[wave][(staged * R + c) * kTile + 8 * g];
        st16(at, __builtin_bit_cast(u32x4, f32x4{raw[0][0], raw[0][1], raw[0][2], raw[0][3]}));
        st16(at + 4, __builtin_bit_cast(u32x4, f32x4{raw[0][4], raw[0][5], raw[0][6], raw[0][7]}));
      }
      if (++staged == stage_tiles || n0 == last) flush_scores(n0);
    } else if constexpr (SCORES) {
      const float* out = a.raw + ((int64_t)(b * a.hkv + kvh) * a.raw_tiles + n0 / kTile) * R * kTile;
      const auto r = make_rsrc(out, (uint32_t)R * kTile * 4);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int at = ((r0 + 16 * t + c) * kTile + 8 * g) * 4;
#pragma unroll
        for (int i = 0; i < 8; i += 4)
          __builtin_amdgcn_raw_buffer_store_b128(
              __builtin_bit_cast(u32x4, f32x4{raw[t][i], raw[t][i + 1], raw[t][i + 2], raw[t][i + 3]}), r, at + 4 * i, 0, 0);
      }
    }
  };
  // the tile's pairs through LDS: each lane converts one, every lane reads eight keys'
  auto store_pair = [&](uint32_t w) __attribute__((always_inline)) {
    if constexpr (I4) {
      const float sc = lo_f32<F16>(w), z = hi_f32<F16>(w);
      const f32x2 v = {16.f * sc * (vlane ? 1.f : cs), vlane ? __builtin_fmaf(7.5f, sc, z) : z * cs};
      *(f32x2*)&pairs[wave][2 * lane] = v;
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  };

  if constexpr (!REFILL) {
    // The next tile is in flight while one is worked on (two or three ahead, or two tiles a step at D = 64, gain nothing
    // or spill).
    auto step = [&](Tile& cur, Tile& next) __attribute__((always_inline)) {
      store_pair(cur.pair);
      if (n0 + STEP <= last) load_tile(n0 + STEP, next);
      f32x4 acc[RT][2];
      product_k(cur, acc);
      product_v(cur, acc, n0);
      store_scores(n0);
      n0 += STEP;
    };
    while (n0 <= last) {
      step(tiles[0], tiles[1]);
      if (n0 > last) break;
      step(tiles[1], tiles[0]);
    }
  } else {
    // K's registers are refilled once its product has read them, V's likewise
    Tile& t = tiles[0];
    for (; n0 <= last; n0 += STEP) {
      f32x4 acc[RT][2];
      store_pair(t.pair);
      product_k(t, acc);
      if (n0 + STEP <= last) load_k(n0 + STEP, t);
      product_v(t, acc, n0);
      if (n0 + STEP <= last) load_v(n0 + STEP, t);
      store_scores(n0);
    }
  }

  if constexpr (QLDS) __syncthreads();  // every wave has read its Q
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

// What follows the partitions' partials: blocks below a.merge_blocks merge a row's partials into its output, the others
// turn scores into weights.  Both start from the partitions' (max, sum), so neither waits for the other: one launch.
// For up to kMergeSplits partitions (more: splitk_combine_kernel, which spreads a row's partials over a workgroup, and
// then this kernel with the log-sum-exps that it wrote: 5 us more in all for 32 x 8 heads x 8 rows that score 8191 keys).
constexpr int kMergeSplits = 16;
constexpr int kFinishRows = 512;  // rows whose log-sum-exps a block holds at a time

// D/4 lanes a row, rows of a block one after another; log-sum-exp merge as splitk_combine_kernel:
//   m = max_s m_s,  w_s = 2^(m_s - m) l_s,  O = sum_s w_s O_s / sum_s w_s
template <int D, class E>
__device__ __forceinline__ void merge_rows(const FinishArgs& a) {
  constexpr int LPR = D / 4, CH = 4;
  constexpr float NEG_INF = -__builtin_inff();
  const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + (int)threadIdx.x / LPR;
  if (row >= a.rows) return;
  const int d = (int)threadIdx.x % LPR * 4;
  const uint32_t bh = (uint32_t)row / (uint32_t)a.nq, qi = (uint32_t)row - bh * (uint32_t)a.nq;
  const uint32_t b = bh / (uint32_t)a.hq, hq = bh - b * (uint32_t)a.hq;
  int S = a.n_split;  // partitions that start below the sequence's end: the others were not written
  if (a.seqlens_k != nullptr) S = min(S, (min(max(a.seqlens_k[b], 0), a.nk) + a.split_len - 1) / a.split_len);
  const float* ml = a.ml + row * a.n_split * 2;
  const float* part = a.part + row * a.n_split * D + d;
  float m = NEG_INF, l = 0.f;
  f32x4 acc = {};
  for (int s0 = 0; s0 < S; s0 += CH) {
    f32x2 st[CH];
    f32x4 o[CH];
#pragma unroll
    for (int u = 0; u < CH; ++u) {  // past the last: the last again, which weighs 0
      const int s = min(s0 + u, S - 1);
      st[u] = __builtin_bit_cast(f32x2, ld8(ml + 2 * s));
      o[u] = __builtin_bit_cast(f32x4, ld16(part + s * D));
      if (s0 + u >= S) st[u] = f32x2{NEG_INF, 0.f};
    }
    float m_new = m;
#pragma unroll
    for (int u = 0; u < CH; ++u) m_new = fmaxf(m_new, st[u][0]);
    const float ref = m_new == NEG_INF ? 0.f : m_new, alpha = fast_exp2(m - ref);
    l *= alpha;
    acc *= alpha;
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      const float w = fast_exp2(st[u][0] - ref) * st[u][1];
      l += w;
      acc += s0 + u < S ? w * o[u] : f32x4{};
    }
    m = m_new;
  }
  const float l_safe = l == 0.f ? 1.f : l, inv = 1.f / l_safe;
  if (a.lse != nullptr && d == 0) a.lse[b * a.slb + hq * a.slh + qi] = (m + __log2f(l_safe)) * kLn2;
  st8((uint16_t*)a.o + b * a.sob + hq * a.soh + qi * a.son + d,
      u32x2{pack2<E>(acc[0] * inv, acc[1] * inv), pack2<E>(acc[2] * inv, acc[3] * inv)});
}

// score_j = before_j + sum over the rows of 2^(s_rj - lse2_r), for the keys that a row sees.  Four keys a lane; NW waves
// share 256 keys and take every NW-th row each (their sums are added in order), and a block has 4 / NW such sets.  16
// waves from 64 rows on (8 heads x 128 rows, 8191 keys: 12 us, one wave 34), else one (16 x 8 heads x 4 rows, 16384
// keys: 12 us, sixteen 116).
template <int NW>
__device__ __forceinline__ void finish_scores(const FinishArgs& a) {
  constexpr int THREADS = NW <= 4 ? 256 : NW * 64, SETS = THREADS / 64 / NW;
  constexpr float NEG_INF = -__builtin_inff();
  __shared__ float lse2[kFinishRows];
  __shared__ __align__(16) float sums[NW > 1 ? NW : 1][NW > 1 ? 256 : 4];
  const uint32_t blk = blockIdx.x - (uint32_t)a.merge_blocks;
  const int bh = (int)(blk / (uint32_t)a.chunks), b = bh / a.hkv, kvh = bh - b * a.hkv;
  const int seq_k = a.seqlens_k != nullptr ? min(max(__builtin_amdgcn_readfirstlane(a.seqlens_k[b]), 0), a.nk) : a.nk;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int block0 = (int)(blk - (uint32_t)bh * (uint32_t)a.chunks) * (256 * SETS);
  const int j0 = block0 + wave / NW * 256, j = j0 + 4 * lane;
  const int R = a.group * a.nq, offset = seq_k - a.nq, w0 = wave % NW;
  const int S = a.seqlens_k != nullptr ? min(a.n_split, (seq_k + a.split_len - 1) / a.split_len) : a.n_split;
  const int64_t prow = ((int64_t)b * a.hq + kvh * a.group) * a.nq;  // (row r of the group: prow + r)
  const float* raw = a.raw + ((int64_t)bh * a.raw_tiles + j / kTile) * R * kTile + j % kTile;
  // the first rows' scores are on their way while their log-sum-exps are formed
  constexpr int PRE = 8;
  const bool masked = a.causal && a.nq > 1;  // (one query sees every key)
  auto end_of = [&](int r) __attribute__((always_inline)) { return masked ? min(seq_k, r % a.nq + offset + 1) : seq_k; };
  f32x4 w = {}, first[PRE];
#pragma unroll
  for (int u = 0; u < PRE; ++u) {
    const int r = w0 + u * NW;
    first[u] = f32x4{};
    if (r < R && j < end_of(r)) first[u] = __builtin_bit_cast(f32x4, ld16(raw + r * kTile));
  }
  for (int r0 = 0; r0 < R && block0 < seq_k; r0 += kFinishRows) {
    const int rows = min(kFinishRows, R - r0);
    if (r0 > 0) __syncthreads();
    for (int r = (int)threadIdx.x; r < rows; r += THREADS) {
      float x;
      if (a.use_lse) {
        const int gi = (r0 + r) / a.nq;
        x = a.lse[b * a.slb + (kvh * a.group + gi) * a.slh + (r0 + r - gi * a.nq)] * kLog2e;
      } else {
        const float* ml = a.ml + (prow + r0 + r) * a.n_split * 2;
        f32x2 st[kMergeSplits];  // all loads in flight
#pragma unroll
        for (int s = 0; s < kMergeSplits; ++s) st[s] = s < S ? __builtin_bit_cast(f32x2, ld8(ml + 2 * s)) : f32x2{NEG_INF, 0.f};
        float m = NEG_INF, l = 0.f;
#pragma unroll
        for (int s = 0; s < kMergeSplits; ++s) m = fmaxf(m, st[s][0]);
        const float ref = m == NEG_INF ? 0.f : m;
#pragma unroll
        for (int s = 0; s < kMergeSplits; ++s) l += fast_exp2(st[s][0] - ref) * st[s][1];
        x = m + __log2f(l == 0.f ? 1.f : l);
      }
      lse2[r] = x;
    }
    __syncthreads();
    auto add = [&](int r, const f32x4& s) __attribute__((always_inline)) {  // r: below this chunk's rows
      const float l2 = lse2[r];
      const int end = l2 == NEG_INF ? 0 : end_of(r0 + r);  // (-inf: every key of the row scores -inf)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] += j + i < end ? fast_exp2(s[i] - l2) : 0.f;
    };
    int done = 0;
    if (r0 == 0) {
#pragma unroll
      for (int u = 0; u < PRE; ++u) {
        if (w0 + u * NW < rows) add(w0 + u * NW, first[u]);
      }
      done = PRE * NW;
    }
    if (j0 < seq_k) {
#pragma unroll 8
      for (int r = done + w0; r < rows; r += NW) {
        f32x4 s = {};
        if (j < end_of(r0 + r)) s = __builtin_bit_cast(f32x4, ld16(raw + (r0 + r) * kTile));
        add(r, s);
      }
    }
  }
  const float* in = a.in != nullptr ? a.in + b * a.sib + kvh * a.sih : nullptr;
  float* out = a.out + b * a.sob_s + kvh * a.soh_s;
  if constexpr (NW > 1) {
    *(f32x4*)&sums[wave][4 * lane] = w;
    __syncthreads();
    const int t = (int)threadIdx.x, key = block0 + t;
    if (t >= 256 || key >= a.nk) return;
    float x = sums[0][t];
#pragma unroll
    for (int i = 1; i < NW; ++i) x += sums[i][t];
    out[key] = in != nullptr ? x + in[key] : x;
  } else if (a.wide && j + 4 <= a.nk) {
    if (in != nullptr) w += __builtin_bit_cast(f32x4, ld16(in + j));
    st16(out + j, __builtin_bit_cast(u32x4, w));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (j + i < a.nk) out[j + i] = in != nullptr ? w[i] + in[j + i] : w[i];
    }
  }
}

template <int D, class E, int NW>
__global__ void __launch_bounds__(NW <= 4 ? 256 : NW * 64) cache_finish_kernel(const FinishArgs a) {
  if ((int)blockIdx.x < a.merge_blocks) {
    if (threadIdx.x < 256) merge_rows<D, E>(a);
  } else {
    finish_scores<NW>(a);
  }
}

template <int D, class E>
hipError_t launch_finish(FinishArgs a, bool merge, bool scores, hipStream_t stream, const char** err) {
  const int R = a.group * a.nq, nw = R >= 64 ? 16 : 1, keys = nw == 16 ? 256 : 1024;
  a.chunks = (a.nk + keys - 1) / keys;
  const int64_t mb = merge ? (a.rows + 1024 / D - 1) / (1024 / D) : 0, fb = scores ? (int64_t)a.batch * a.hkv * a.chunks : 0;
  if (mb + fb > INT32_MAX) {
    *err = "grid too large";
    return hipErrorInvalidConfiguration;
  }
  a.merge_blocks = (int32_t)mb;
  if (mb + fb == 0) return hipSuccess;
  if (nw == 16 && scores) {
    hipLaunchKernelGGL((cache_finish_kernel<D, E, 16>), dim3((unsigned)(mb + fb)), dim3(1024), 0, stream, a);
  } else {
    hipLaunchKernelGGL((cache_finish_kernel<D, E, 1>), dim3((unsigned)(mb + fb)), dim3(256), 0, stream, a);
  }
  return hipGetLastError();
}

template <int D, class E, bool I4, bool PAGED, bool SCORES>
hipError_t launch_rows(const CacheArgs& a, int rt, hipStream_t stream) {
  if (rt == 1) {
    hipLaunchKernelGGL((attn_cache_kernel<D, E, I4, PAGED, SCORES, 1>), dim3((unsigned)a.total), dim3(kCacheWaves * 64),
                       0, stream, a);
  } else if (rt == 2) {
    hipLaunchKernelGGL((attn_cache_kernel<D, E, I4, PAGED, SCORES, 2>), dim3((unsigned)a.total), dim3(kCacheWaves * 64),
                       0, stream, a);
  } else if constexpr (D != 256) {
    hipLaunchKernelGGL((attn_cache_kernel<D, E, I4, PAGED, SCORES, 4>), dim3((unsigned)a.total), dim3(kCacheWaves * 64),
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

int raw_tiles(const fa_cache_params& p) { return (p.seqlen_k + kTile - 1) / kTile; }

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

int splits(const fa_cache_params& p, int split_len) {
  return p.seqlen_k > 0 ? (p.seqlen_k + split_len - 1) / split_len : 1;
}

// Row blocks of 16 that a workgroup takes together.
int row_tiles(const fa_cache_params& p) {
  const int64_t rows = (int64_t)(p.heads_q / p.heads_kv) * p.seqlen_q;
  return rows <= 16 ? 1 : rows <= 32 || p.head_dim == 256 ? 2 : 4;
}

// Workgroups of attn_cache_kernel.
int64_t workgroups(const fa_cache_params& p, int n_split) {
  const int64_t items = (int64_t)p.batch * p.heads_kv * n_split, rows = (int64_t)(p.heads_q / p.heads_kv) * p.seqlen_q;
  const int block = 16 * row_tiles(p);
  return (p.seqlens_k != nullptr ? (items + 7) / 8 * 8 : items) * ((rows + block - 1) / block);
}

}  // namespace

const char* cache_refusal(const fa_cache_params& p, int32_t split_len) {
  if (p.block_table != nullptr && ((int64_t)split_len - 1) / p.page_size + 2 > kMaxSlots)
    return "split_len too long for the page size: a partition may span at most 258 pages";
  if ((int64_t)p.batch * p.heads_q * p.seqlen_q > INT32_MAX || workgroups(p, splits(p, split_len)) > INT32_MAX)
    return "grid too large";
  // (a tile's scores are addressed by 32-bit byte offsets: 128 a row)
  if (p.scores_out != nullptr && (int64_t)(p.heads_q / p.heads_kv) * p.seqlen_q > (1 << 23))
    return "scores are formed for at most 2^23 (q-head, query) rows a kv-head";
  return nullptr;
}

size_t cache_workspace_bytes(const fa_cache_params& p, int32_t split_len) {
  size_t need = align16(fa_splitk_workspace_bytes(p.batch, p.heads_q, p.seqlen_q, p.head_dim, splits(p, split_len)));
  if (p.scores_out != nullptr) {
    const size_t rows = (size_t)p.batch * p.heads_q * p.seqlen_q;
    need += align16(rows * sizeof(float)) + rows * (size_t)raw_tiles(p) * kTile * sizeof(float);
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
  }
  const int rows = a.group * p.seqlen_q, rt = row_tiles(p);
  a.n_rowblk = (rows + 16 * rt - 1) / (16 * rt);
  const int64_t items = (int64_t)p.batch * p.heads_kv * S, out_rows = (int64_t)p.batch * p.heads_q * p.seqlen_q;
  const int64_t total = workgroups(p, S);
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
    a.raw_tiles = raw_tiles(p);
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

  const bool merge = S <= kMergeSplits;
  if (!merge) {
    CombineArgs c{};
    c.opart = a.part, c.ml = a.ml, c.o = p.o;
    c.sob = p.o_stride_b, c.soh = p.o_stride_h, c.son = p.o_stride_n;
    c.lse = lse, c.slb = slb, c.slh = slh;
    c.hq = p.heads_q, c.group = a.group, c.nq = p.seqlen_q, c.n_split = S;
    c.seqlens_k = p.seqlens_k, c.nk = p.seqlen_k, c.split_len = split_len;
    const fa_status st = run_combine(c, p.head_dim, bf, out_rows, stream, err);
    if (st != FA_OK) return st;
  }
  FinishArgs f{};
  f.part = a.part, f.ml = a.ml, f.o = p.o;
  f.sob = p.o_stride_b, f.soh = p.o_stride_h, f.son = p.o_stride_n;
  f.raw = a.raw, f.raw_tiles = a.raw_tiles;
  f.lse = merge ? p.lse : lse, f.slb = slb, f.slh = slh;
  f.use_lse = merge ? 0 : 1;
  f.in = p.scores_in, f.sib = p.scores_in_stride_b, f.sih = p.scores_in_stride_h;
  f.out = p.scores_out, f.sob_s = p.scores_out_stride_b, f.soh_s = p.scores_out_stride_h;
  f.wide = (((uintptr_t)f.in | (uintptr_t)f.out) % 16 == 0 && (f.sib | f.sih | f.sob_s | f.soh_s) % 4 == 0) ? 1 : 0;
  f.seqlens_k = p.seqlens_k;
  f.rows = out_rows;
  f.batch = p.batch, f.hq = p.heads_q, f.hkv = p.heads_kv, f.group = a.group, f.nq = p.seqlen_q, f.nk = p.seqlen_k;
  f.causal = a.causal, f.n_split = S, f.split_len = split_len;
  if (p.head_dim == 64) {
    e = bf ? launch_finish<64, BF16>(f, merge, scores, stream, err) : launch_finish<64, F16>(f, merge, scores, stream, err);
  } else if (p.head_dim == 128) {
    e = bf ? launch_finish<128, BF16>(f, merge, scores, stream, err) : launch_finish<128, F16>(f, merge, scores, stream, err);
  } else {
    e = bf ? launch_finish<256, BF16>(f, merge, scores, stream, err) : launch_finish<256, F16>(f, merge, scores, stream, err);
  }
  return hip_status(e, err);
}

}  // namespace fa
