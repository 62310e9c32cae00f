// Eviction from a K/V cache by accumulated attention weight: which keys stay, and their rows moved together.
//
// Per (sequence, kv-head), with n keys in the cache and room for `keep`: all keys where n <= keep; else the last
// `recent` ones and, of the others, the keep - recent with the highest scores (equal scores: the lower index; a NaN
// counts as the highest, -0 as 0), in their order in the cache.
//
//   * evict_select_kernel: one workgroup a (sequence, kv-head).  The threshold is found digit by digit: scores map to
//     unsigned integers of the same order, and three passes each count the digits of the candidates that share the
//     digits found so far.  Integer counts in LDS: the result does not depend on the order of the additions.  A last
//     pass writes the indices in order (the candidates above the threshold and the first of those equal to it).
//   * gather_rows_kernel: the scores and the rows of up to eight tensors in one launch; a thread copies units of the widest
//     power of two (16 bytes at most) that a tensor's rows, strides and addresses allow.  HBM-bound: 16 x 8 heads, 4096
//     of 8192 keys with 4-bit rows of D=128, 33 us (161 MB moved: 4.9 TB/s); 8 heads, 16384 of 65536 with bf16 rows of
//     D=128, 27 us (139 MB: 5.1 TB/s).  A branch around each load, so that one waits for another: 45 and 31 us.
#include "fa_device.hpp"
#include "fa_internal.hpp"

namespace fa {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kItems = 4;
constexpr int kCopies = 4;

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // rows of scores start at any float

// Unsigned integers in the order of the scores: NaN above +inf, -0 equal to 0.  Never 0 (-inf gives 0x007fffff).
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  if (x != x) return 0xffffffffu;
  if (u == 0x80000000u) return 0x80000000u;
  return (u >> 31) ? ~u : u | 0x80000000u;
}

// Inclusive sums over the lanes up to this one: of its 16 lanes by DPP moves, and of the wave by adding the last lane
// of each 16 (then of each 32) to those behind it.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t x) {
  return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t row_scan(uint32_t x) {
  return dpp_add<0x118, 0xf>(dpp_add<0x114, 0xf>(dpp_add<0x112, 0xf>(dpp_add<0x111, 0xf>(x))));  // row_shr:1, 2, 4, 8
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  return dpp_add<0x143, 0xc>(dpp_add<0x142, 0xa>(row_scan(x)));  // row_bcast:15 into rows 1 and 3, :31 into 2 and 3
}

// A thread holds the keys of four candidates of each of CH chunks of 4096 in registers, all loads in flight; up to
// CH * 4096 candidates are read once, more again in every pass.  Two chunks where they hold every key (16 x 8 heads x
// 8192 keys: 12 us, with eight 23), else eight (8 heads x 65536 keys: 47 us; two chunks 53, sixteen do not fit the 128
// registers of 1024 threads and spill, 58).  Digits of 11, 11 and 10 bits: the first already tells a quarter of an octave
// apart; the candidates that share it are gathered in LDS if they fit, and the others count those.  One workgroup a head:
// bound by its own instructions and waits, not by memory.
template <int CH>
__global__ void __launch_bounds__(kThreads) evict_select_kernel(const EvictArgs a) {
  constexpr int CHUNK = kThreads * kItems, SPAN = CH * CHUNK;
  constexpr int BINS = 2048, LIST = 4096;
  constexpr int DPT = BINS / kThreads;  // digits a thread
  __shared__ __align__(16) uint32_t hist[BINS * kCopies];
  __shared__ uint32_t list[LIST];
  // this pass's digit, how many are still wanted among its candidates, the list's length, the digit's candidates
  __shared__ uint32_t found[4];
  __shared__ uint32_t wave_sum[CH * kWaves];

  const int bh = (int)blockIdx.x, b = bh / a.h, h = bh - b * a.h;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = a.seqlens_k != nullptr ? min(max(a.seqlens_k[b], 0), a.nk) : a.nk;
  const float* s = a.scores + b * a.ssb + h * a.ssh;
  int32_t* index = a.index + (int64_t)bh * a.keep;
  if (h == 0 && tid == 0) a.seqlens_out[b] = min(n, a.keep);

  if (n <= a.keep) {
    for (int j = tid; j < a.keep; j += kThreads) index[j] = j < n ? j : -1;
    return;
  }
  const int old = n - a.recent, want = a.keep - a.recent;  // 0 <= recent <= keep < n
  for (int j = tid; j < a.recent; j += kThreads) index[want + j] = old + j;
  if (want == 0) return;

  // keys of this thread's candidates from `base` on; past the last: 0, which no score's key is
  u32x4 held[CH];
  auto load = [&](int base) __attribute__((always_inline)) {
    f32x4 raw[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int j = base + i * CHUNK + tid * kItems;
      raw[i] = f32x4{};
      if (j + kItems <= old) {
        const f32x4u v = *(const f32x4u*)(s + j);
        raw[i] = f32x4{v[0], v[1], v[2], v[3]};
      } else {
#pragma unroll
        for (int e = 0; e < kItems; ++e) {
          if (j + e < old) raw[i][e] = s[j + e];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int j = base + i * CHUNK + tid * kItems;
#pragma unroll
      for (int e = 0; e < kItems; ++e) held[i][e] = j + e < old ? order_key(raw[i][e]) : 0u;
    }
  };
  if (old <= SPAN) load(0);

  // ---- the key of rank `want` among the candidates [0, old) ------------------------------------------------
  // (the 0s past the last are counted as the lowest digit of the first pass, which no key has and no rank reaches)
  uint32_t prefix = 0, rank = (uint32_t)want, listed = 0;  // listed: candidates in `list`, 0 while it is not made
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digits = pass == 2 ? 1023u : 2047u, mask = pass == 0 ? 0u : ~0u << (shift + (pass == 1 ? 11 : 10));
    for (int i = tid * 4; i < BINS * kCopies; i += kThreads * 4) st16(&hist[i], u32x4{});
    if (tid == 0) found[2] = 0;
    __syncthreads();
    uint32_t* mine = hist + (lane & (kCopies - 1));
    if (pass == 1 && listed != 0) {
      // the candidates of the first digit, in any order: the passes left count these alone
      for (int base = 0; base < old; base += SPAN) {
        if (old > SPAN) load(base);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
#pragma unroll
          for (int e = 0; e < kItems; ++e) {
            const bool in = (held[i][e] & mask) == prefix;
            const uint64_t who = __builtin_amdgcn_ballot_w64(in);
            if (who == 0) continue;
            uint32_t at = 0;
            if (lane == 0) at = atomicAdd(&found[2], (uint32_t)__popcll(who));
            at = __builtin_amdgcn_readfirstlane(at) +
                 __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
            if (in) list[at] = held[i][e];
          }
        }
      }
      __syncthreads();
    }
    auto count = [&](uint32_t k) __attribute__((always_inline)) {
      if ((k & mask) == prefix) atomicAdd(&mine[((k >> shift) & digits) * kCopies], 1u);
    };
    if (listed != 0) {
      for (uint32_t i = (uint32_t)tid; i < listed; i += kThreads) count(list[i]);
    } else {
      for (int base = 0; base < old; base += SPAN) {
        if (old > SPAN) load(base);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
#pragma unroll
          for (int e = 0; e < kItems; ++e) count(held[i][e]);
        }
      }
    }
    __syncthreads();
    // thread t: the counts of DPT digits from the highest down, then how many candidates lie above them
    const int d = BINS - 1 - DPT * tid;
    uint32_t c[DPT], sum = 0;
#pragma unroll
    for (int i = 0; i < DPT; ++i) {
      c[i] = 0;
#pragma unroll
      for (int u = 0; u < kCopies; u += 4) {
        const u32x4 t = ld16(&hist[(d - i) * kCopies + u]);
        c[i] += t[0] + t[1] + t[2] + t[3];
      }
      sum += c[i];
    }
    const uint32_t upto = wave_scan(sum);
    if (lane == 63) wave_sum[wave] = upto;
    __syncthreads();
    uint32_t over = upto - sum;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) over += w < wave ? wave_sum[w] : 0u;
#pragma unroll
    for (int i = 0; i < DPT; ++i) {
      if (over < rank && over + c[i] >= rank) {  // one thread and digit: its candidates hold the one of this rank
        found[0] = (uint32_t)(d - i);
        found[1] = rank - over;
        found[3] = c[i];
      }
      over += c[i];
    }
    __syncthreads();
    prefix |= found[0] << shift;
    rank = found[1];
    if (pass == 0 && found[3] <= LIST) listed = found[3];
  }

  // ---- indices in order: keys above `prefix`, and the first `rank` equal to it ------------------------------
  auto flags = [&](const u32x4& k, uint32_t(&flag)[kItems]) __attribute__((always_inline)) {
    uint32_t sum = 0;  // above in the low half, equal in the high half (a chunk holds 4096 at most)
#pragma unroll
    for (int e = 0; e < kItems; ++e) sum += flag[e] = k[e] > prefix ? 1u : k[e] == prefix ? 0x10000u : 0u;
    return sum;
  };
  uint32_t above = 0, equal = 0;  // before `base`
  for (int base = 0; base < old; base += SPAN) {
    if (old > SPAN) load(base);
    uint32_t flag[kItems];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const uint32_t upto = wave_scan(flags(held[i], flag));
      if (lane == 63) wave_sum[i * kWaves + wave] = upto;
    }
    __syncthreads();
    __asm__("" : "+v"(prefix));  // the flags again: kept from above they would take as many registers as the keys
    // lane 16q + w: chunk 4p + q's sums of the waves up to w
    static_assert(kWaves == 16, "a chunk's waves are 16 lanes");
    uint32_t scan[(CH + 3) / 4];
#pragma unroll
    for (int p = 0; p < (CH + 3) / 4; ++p) scan[p] = row_scan(4 * p + lane / 16 < CH ? wave_sum[p * 64 + lane] : 0u);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int j = base + i * CHUNK + tid * kItems, first = i % 4 * 16;
      const uint32_t sum = flags(held[i], flag);
      const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)scan[i / 4], first + 15);
      uint32_t before = wave_scan(sum) - sum;
      if (wave > 0) before += (uint32_t)__builtin_amdgcn_readlane((int)scan[i / 4], first + wave - 1);
      uint32_t na = above + (before & 0xffffu), ne = equal + (before >> 16);
#pragma unroll
      for (int e = 0; e < kItems; ++e) {
        if (flag[e] == 1u || (flag[e] != 0u && ne < rank)) index[na + min(ne, rank)] = j + e;
        na += flag[e] & 0xffffu;
        ne += flag[e] >> 16;
      }
      above += all & 0xffffu;
      equal += all >> 16;
    }
    if (base + SPAN < old) __syncthreads();  // the next span's sums replace these
  }
}

template <class U>
__device__ __forceinline__ void gather_units(const EvictTensor& t, const EvictArgs& a, int bh) {
  constexpr int STEP = 4;
  const int b = bh / a.h, h = bh - b * a.h;
  const char* src = (const char*)t.src + b * t.sb + h * t.sh;
  char* dst = (char*)t.dst + b * t.db + h * t.dh;
  const int32_t* index = a.index + (int64_t)bh * a.keep;
  const uint32_t units = (uint32_t)t.units, all = (uint32_t)a.keep * units;  // < 2^31 (host)
  const uint32_t u0 = (uint32_t)(blockIdx.x % (uint32_t)a.chunks) * (256 * STEP) + threadIdx.x;
  if (u0 - threadIdx.x >= all) return;  // (another tensor's rows have more units)
  // No branch around the loads (units past the last are the last one's, and -1 reads row 0, which a tensor with rows to
  // fill has), so all of a kind are in flight together.
  uint32_t r[STEP], c[STEP];
  int j[STEP];
#pragma unroll
  for (int i = 0; i < STEP; ++i) {
    const uint32_t u = min(u0 + 256 * i, all - 1);
    r[i] = t.shift >= 0 ? u >> t.shift : u / units, c[i] = u - r[i] * units;
    j[i] = index[r[i]];
  }
  U v[STEP];
#pragma unroll
  for (int i = 0; i < STEP; ++i) v[i] = *(const U*)(src + max(j[i], 0) * t.sn + c[i] * sizeof(U));
#pragma unroll
  for (int i = 0; i < STEP; ++i) {
    const U x = j[i] >= 0 ? v[i] : U{};
    if (u0 + 256 * i < all) *(U*)(dst + r[i] * t.dn + c[i] * sizeof(U)) = x;
  }
}

// blockIdx.y: tensor; blockIdx.x: (sequence and kv-head, chunk of its kept rows' units)
__global__ void __launch_bounds__(256) gather_rows_kernel(const EvictArgs a) {
  const EvictTensor& t = a.tensors[blockIdx.y];
  const int bh = (int)(blockIdx.x / (uint32_t)a.chunks);
  switch (t.unit) {  // uniform
    case 16: return gather_units<u32x4>(t, a, bh);
    case 8: return gather_units<u32x2>(t, a, bh);
    case 4: return gather_units<uint32_t>(t, a, bh);
    case 2: return gather_units<uint16_t>(t, a, bh);
    default: return gather_units<uint8_t>(t, a, bh);
  }
}

}  // namespace

fa_status run_evict(const fa_evict_params& p, hipStream_t stream, const char** err) {
  EvictArgs a{};
  a.scores = p.scores;
  a.ssb = p.scores_stride_b;
  a.ssh = p.scores_stride_h;
  a.seqlens_k = p.seqlens_k;
  a.index = p.index;
  a.seqlens_out = p.seqlens_out;
  a.h = p.heads;
  a.nk = p.seqlen;
  a.keep = p.keep;
  a.recent = p.recent;
  const int64_t bh = (int64_t)p.batch * p.heads;
  int64_t units = 0;  // most of any tensor, per (sequence, kv-head)
  auto add = [&](EvictTensor& g, const fa_evict_tensor& t) {
    const uint64_t bits = (uint64_t)(uintptr_t)t.src | (uint64_t)(uintptr_t)t.dst | (uint64_t)t.row_bytes |
                          (uint64_t)t.src_stride_b | (uint64_t)t.src_stride_h | (uint64_t)t.src_stride_n |
                          (uint64_t)t.dst_stride_b | (uint64_t)t.dst_stride_h | (uint64_t)t.dst_stride_n | 16u;
    const int64_t unit = (int64_t)(bits & (~bits + 1)), n = t.row_bytes / unit;  // unit: the lowest set bit
    g = EvictTensor{t.src, t.dst, t.src_stride_b, t.src_stride_h, t.src_stride_n, t.dst_stride_b, t.dst_stride_h,
                    t.dst_stride_n, (int32_t)unit, (int32_t)n, -1};
    for (int s = 0; s < 31; ++s) {
      if ((int64_t{1} << s) == n) g.shift = s;
    }
    const int64_t all = n <= INT32_MAX ? (int64_t)p.keep * n : INT64_MAX;
    units = units > all ? units : all;
  };
  const int64_t row = (int64_t)p.keep * 4;
  const fa_evict_tensor scores = {p.scores, p.scores_out, p.scores_stride_b * 4, p.scores_stride_h * 4, 4,
                                  p.heads * row, row, 4, 4};
  add(a.tensors[0], scores);
  for (int i = 0; i < p.num_tensors; ++i) add(a.tensors[i + 1], p.tensors[i]);
  if (units > INT32_MAX - 1024 || bh > INT32_MAX || bh * ((units + 1023) / 1024) > INT32_MAX) {
    *err = "grid too large";
    return FA_ERR_UNSUPPORTED;
  }
  a.chunks = (int32_t)((units + 1023) / 1024);
  auto select = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)bh), dim3(kThreads), 0, stream, a); };
  a.nk <= 2 * kThreads * kItems ? select(evict_select_kernel<2>) : select(evict_select_kernel<8>);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.chunks == 0) return hip_status(e, err);
  hipLaunchKernelGGL(gather_rows_kernel, dim3((unsigned)(bh * a.chunks), (unsigned)p.num_tensors + 1), dim3(256), 0, stream,
                     a);
  return hip_status(hipGetLastError(), err);
}

}  // namespace fa
