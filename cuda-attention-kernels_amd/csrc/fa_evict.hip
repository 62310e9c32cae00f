// Eviction from a K/V cache by accumulated attention weight: which keys stay, and their rows moved together.
//
// Per (sequence, kv-head), with n keys in the cache and room for `keep`: all keys where n <= keep; else the last
// `recent` ones and, of the others, the keep - recent with the highest scores (equal scores: the lower index; a NaN
// counts as the highest, -0 as 0), in their order in the cache.
//
// The threshold is found digit by digit: scores map to unsigned integers of the same order, and digits of 11, 11 and 10
// bits are counted among the candidates that share the digits found so far.  Integer counts: the result does not depend
// on the order of the additions.  A last pass writes the indices in order (the candidates above the threshold and the
// first of those equal to it).
//
//   * evict_select_kernel: up to 8192 keys, one workgroup a (sequence, kv-head), which holds them in registers.
//   * evict_count_kernel, evict_list_kernel, evict_index_kernel: more keys, up to 16 workgroups a (sequence, kv-head), each
//     with a range of them.  Bound by vector instructions (about 80 a key and wave), so the work is spread: 8 heads x
//     65536 keys took one workgroup each 49 us, and take the three launches 25.  Every group reads the whole list of the
//     keys that share the threshold's first digit, so where most do (all scores equal, or most of them 0) it takes 67.
//   * gather_rows_kernel: the scores and the rows of up to eight tensors in one launch; a thread copies units of the widest
//     power of two (16 bytes at most) that a tensor's rows, strides and addresses allow.  HBM-bound: 16 x 8 heads, 4096
//     of 8192 keys with 4-bit rows of D=128, 33 us (161 MB moved: 4.9 TB/s); 8 heads, 16384 of 65536 with bf16 rows of
//     D=128, 27 us (139 MB: 5.1 TB/s).  A branch around each load, so that one waits for another: 45 and 31 us.
#include "fa_device.hpp"
#include "fa_internal.hpp"

namespace fa {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kItems = 4;
constexpr int kChunk = kThreads * kItems, kHeld = 2;  // a thread holds four keys of each of two chunks
constexpr int kSpan = kHeld * kChunk, kMaxGroups = 16;
constexpr int kBins = 2048, kCopies = 4, kDigits = kBins / kThreads;  // (digits a thread looks after)
constexpr int kShift[3] = {21, 10, 0};

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

// The candidates [0, old) of a (sequence, kv-head): all but the `recent` last of its n keys.
struct Candidates {
  int n, old, want;
  const float* s;
  int32_t* index;
  __device__ __forceinline__ Candidates(const EvictArgs& a, int bh) {
    const int b = bh / a.h, h = bh - b * a.h;
    n = a.seqlens_k != nullptr ? min(max(a.seqlens_k[b], 0), a.nk) : a.nk;
    old = n - a.recent, want = a.keep - a.recent;  // 0 <= recent <= keep
    s = a.scores + b * a.ssb + h * a.ssh;
    index = a.index + (int64_t)bh * a.keep;
  }
  // What needs no threshold, by `threads` threads.  True if that was all.
  __device__ __forceinline__ bool simple(const EvictArgs& a, int bh, int tid, int threads) const {
    if (bh % a.h == 0 && tid == 0) a.seqlens_out[bh / a.h] = min(n, a.keep);
    if (n <= a.keep) {
      for (int j = tid; j < a.keep; j += threads) index[j] = j < n ? j : -1;
      return true;
    }
    for (int j = tid; j < a.recent; j += threads) index[want + j] = old + j;
    return want == 0;
  }
  // Keys of this thread's candidates from `base` on, all loads in flight; past the last: 0, which no score's key is.
  __device__ __forceinline__ void load(int base, u32x4 (&held)[kHeld]) const {
    f32x4 raw[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int j = base + i * kChunk + (int)threadIdx.x * kItems;
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
    for (int i = 0; i < kHeld; ++i) {
      const int j = base + i * kChunk + (int)threadIdx.x * kItems;
#pragma unroll
      for (int e = 0; e < kItems; ++e) held[i][e] = j + e < old ? order_key(raw[i][e]) : 0u;
    }
  }
};

struct Shared {
  __align__(16) uint32_t hist[kBins * kCopies];
  uint32_t wave_sum[kHeld * kWaves];
  // the digit found, how many are still wanted among its candidates, how many it has; and two sums
  uint32_t found[5];
};

__device__ __forceinline__ void clear_counts(Shared& sh) {
  for (int i = (int)threadIdx.x * 4; i < kBins * kCopies; i += kThreads * 4) st16(&sh.hist[i], u32x4{});
  __syncthreads();
}

// One candidate of a pass: counted if it shares the digits found before (bits `mask`).
__device__ __forceinline__ void count_key(Shared& sh, uint32_t k, int pass, uint32_t mask, uint32_t prefix) {
  const uint32_t digits = pass == 2 ? 1023u : 2047u;
  if ((k & mask) == prefix) atomicAdd(&sh.hist[((k >> kShift[pass]) & digits) * kCopies + (threadIdx.x & (kCopies - 1))], 1u);
}

// A thread's digits, from the highest down: kBins - 1 - kDigits * thread - i.
__device__ __forceinline__ void counts_of(const Shared& sh, uint32_t (&c)[kDigits]) {
  static_assert(kCopies == 4, "one load a digit");
#pragma unroll
  for (int i = 0; i < kDigits; ++i) {
    const u32x4 t = ld16(&sh.hist[(kBins - 1 - kDigits * (int)threadIdx.x - i) * kCopies]);
    c[i] = t[0] + t[1] + t[2] + t[3];
  }
}

// The digit of the candidate of this rank, from the counts of a thread's digits, into sh.found.  (The 0s past the last
// candidate are counted as the lowest digit of the first pass, which no key has and no rank reaches.)
__device__ __forceinline__ void find_digit(Shared& sh, const uint32_t (&c)[kDigits], uint32_t rank) {
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  uint32_t sum = 0;
#pragma unroll
  for (int i = 0; i < kDigits; ++i) sum += c[i];
  const uint32_t upto = wave_scan(sum);
  if (lane == 63) sh.wave_sum[wave] = upto;
  __syncthreads();
  uint32_t over = upto - sum;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) over += w < wave ? sh.wave_sum[w] : 0u;
#pragma unroll
  for (int i = 0; i < kDigits; ++i) {
    if (over < rank && over + c[i] >= rank) {  // one thread and digit
      sh.found[0] = (uint32_t)(kBins - 1 - kDigits * (int)threadIdx.x - i);
      sh.found[1] = rank - over;
      sh.found[2] = c[i];
    }
    over += c[i];
  }
  __syncthreads();
}

// Above the threshold: 1, equal to it: 0x10000 (a chunk holds 4096 keys).  Their sum over a thread's keys.
__device__ __forceinline__ uint32_t flags_of(const u32x4& k, uint32_t prefix, uint32_t (&flag)[kItems]) {
  uint32_t sum = 0;
#pragma unroll
  for (int e = 0; e < kItems; ++e) sum += flag[e] = k[e] > prefix ? 1u : k[e] == prefix ? 0x10000u : 0u;
  return sum;
}

// The indices of a span's candidates that stay: keys above `prefix`, and of those equal to it the first `rank`.
// above, equal: how many lie before this span, and then before the next.
__device__ __forceinline__ void write_indices(Shared& sh, const u32x4 (&held)[kHeld], int base, uint32_t prefix, uint32_t rank,
                                              int32_t* index, uint32_t& above, uint32_t& equal) {
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t flag[kItems], upto[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    upto[i] = wave_scan(flags_of(held[i], prefix, flag));
    if (lane == 63) sh.wave_sum[i * kWaves + wave] = upto[i];
  }
  __syncthreads();
  // lane 16q + w: chunk q's sums of the waves up to w
  static_assert(kWaves == 16 && kHeld <= 4, "a chunk's waves are 16 lanes");
  const uint32_t scan = row_scan(lane / 16 < kHeld ? sh.wave_sum[lane] : 0u);
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int j = base + i * kChunk + tid * kItems, first = i * 16;
    const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)scan, first + 15);
    uint32_t before = upto[i] - flags_of(held[i], prefix, flag);
    if (wave > 0) before += (uint32_t)__builtin_amdgcn_readlane((int)scan, first + __builtin_amdgcn_readfirstlane(wave) - 1);
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
  __syncthreads();  // (wave_sum is free)
}

// Up to kSpan keys: 16 x 8 heads x 8192 keys in 11 us, bound by its own instructions and waits, not by memory.
__global__ void __launch_bounds__(kThreads) evict_select_kernel(const EvictArgs a) {
  __shared__ Shared sh;
  const int bh = (int)blockIdx.x;
  const Candidates c(a, bh);
  if (c.simple(a, bh, (int)threadIdx.x, kThreads)) return;
  u32x4 held[kHeld];
  c.load(0, held);
  uint32_t prefix = 0, mask = 0, rank = (uint32_t)c.want;
  for (int pass = 0; pass < 3; ++pass) {
    clear_counts(sh);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
#pragma unroll
      for (int e = 0; e < kItems; ++e) count_key(sh, held[i][e], pass, mask, prefix);
    }
    __syncthreads();
    uint32_t counts[kDigits];
    counts_of(sh, counts);
    find_digit(sh, counts, rank);
    prefix |= sh.found[0] << kShift[pass];
    mask = ~0u << kShift[pass];
    rank = sh.found[1];
  }
  uint32_t above = 0, equal = 0;
  write_indices(sh, held, 0, prefix, rank, c.index, above, equal);
}

// More keys: a.groups workgroups a (sequence, kv-head), each with a.group_len keys (whole spans).
struct Group {
  int bh, g, first, end, used;  // its candidates, and how many groups have any
  uint32_t* counts;             // [group][digit] of this (sequence, kv-head)
  uint32_t* list;               // keys of the candidates of the first digit, group by group
  __device__ __forceinline__ Group(const EvictArgs& a) {
    bh = (int)(blockIdx.x / (uint32_t)a.groups), g = (int)(blockIdx.x - (uint32_t)bh * (uint32_t)a.groups);
    counts = a.counts + (int64_t)bh * a.groups * kBins;
    list = a.list + (int64_t)bh * a.nk;
  }
  __device__ __forceinline__ void range(const EvictArgs& a, int old) {
    used = (old + a.group_len - 1) / a.group_len;
    first = min(g * a.group_len, old), end = old - first > a.group_len ? first + a.group_len : old;
  }
  // The first digit of the candidate of this rank (sh.found); `before`: the counts of the groups before this one, of this
  // thread's digits.
  __device__ __forceinline__ void first_digit(Shared& sh, uint32_t rank, uint32_t (&before)[kDigits]) const {
    const int d = kBins - kDigits - kDigits * (int)threadIdx.x;  // the lowest of them
    uint32_t all[kDigits] = {};
    static_assert(kDigits == 2, "one load a group");
    before[0] = before[1] = 0;
#pragma unroll
    for (int i = 0; i < kMaxGroups; ++i) {
      if (i < used) {
        const u32x2 t = __builtin_bit_cast(u32x2, ld8(counts + i * kBins + d));
        all[0] += t[1], all[1] += t[0];
        if (i < g) before[0] += t[1], before[1] += t[0];
      }
    }
    find_digit(sh, all, rank);
  }
};

// The first digit's counts of a group's candidates, and what needs no threshold.
__global__ void __launch_bounds__(kThreads) evict_count_kernel(const EvictArgs a) {
  __shared__ Shared sh;
  Group g(a);
  const Candidates c(a, g.bh);
  if (c.simple(a, g.bh, g.g * kThreads + (int)threadIdx.x, a.groups * kThreads)) return;
  g.range(a, c.old);
  if (g.g >= g.used) return;
  clear_counts(sh);
  for (int base = g.first; base < g.end; base += kSpan) {
    u32x4 held[kHeld];
    c.load(base, held);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
#pragma unroll
      for (int e = 0; e < kItems; ++e) count_key(sh, held[i][e], 0, 0u, 0u);
    }
  }
  __syncthreads();
  uint32_t counts[kDigits];
  counts_of(sh, counts);
  st8(g.counts + g.g * kBins + kBins - kDigits - kDigits * (int)threadIdx.x, u32x2{counts[1], counts[0]});
}

// The keys of a group's candidates that have the first digit, behind those of the groups before it, in any order.
__global__ void __launch_bounds__(kThreads) evict_list_kernel(const EvictArgs a) {
  __shared__ Shared sh;
  Group g(a);
  const Candidates c(a, g.bh);
  if (c.n <= a.keep || c.want == 0) return;
  g.range(a, c.old);
  if (g.g >= g.used) return;
  u32x4 held[kHeld];
  c.load(g.first, held);  // on their way
  uint32_t before[kDigits];
  g.first_digit(sh, (uint32_t)c.want, before);
  const uint32_t digit = sh.found[0];
#pragma unroll
  for (int i = 0; i < kDigits; ++i) {
    if ((uint32_t)(kBins - 1 - kDigits * (int)threadIdx.x - i) == digit) sh.found[3] = before[i];
  }
  __syncthreads();
  const int lane = (int)threadIdx.x & 63;
  for (int base = g.first; base < g.end; base += kSpan) {
    if (base > g.first) c.load(base, held);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
#pragma unroll
      for (int e = 0; e < kItems; ++e) {
        const bool in = held[i][e] >> kShift[0] == digit;
        const uint64_t who = __builtin_amdgcn_ballot_w64(in);
        if (who == 0) continue;
        uint32_t at = 0;
        if (lane == 0) at = atomicAdd(&sh.found[3], (uint32_t)__popcll(who));
        at = __builtin_amdgcn_readfirstlane(at) +
             __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
        if (in) g.list[at] = held[i][e];
      }
    }
  }
}

// The threshold from the list, by every group for itself, and the group's indices.
__global__ void __launch_bounds__(kThreads) evict_index_kernel(const EvictArgs a) {
  __shared__ Shared sh;
  Group g(a);
  const Candidates c(a, g.bh);
  if (c.n <= a.keep || c.want == 0) return;
  g.range(a, c.old);
  if (g.g >= g.used) return;
  u32x4 held[kHeld];
  c.load(g.first, held);
  if (threadIdx.x < 2) sh.found[3 + threadIdx.x] = 0;  // above, listed: of the groups before
  uint32_t before[kDigits];
  g.first_digit(sh, (uint32_t)c.want, before);
  const uint32_t digit = sh.found[0], listed = sh.found[2];
  uint32_t rank = sh.found[1], prefix = digit << kShift[0], mask = ~0u << kShift[0], over = 0;
#pragma unroll
  for (int i = 0; i < kDigits; ++i) {
    const uint32_t d = (uint32_t)(kBins - 1 - kDigits * (int)threadIdx.x - i);
    if (d > digit) over += before[i];
    if (d == digit) sh.found[4] = before[i];
  }
  const int lane = (int)threadIdx.x & 63;
  over = wave_scan(over);
  if (lane == 63 && over != 0) atomicAdd(&sh.found[3], over);
  for (int pass = 1; pass < 3; ++pass) {
    clear_counts(sh);
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < listed; i += kThreads) count_key(sh, g.list[i], pass, mask, prefix);
    __syncthreads();
    uint32_t counts[kDigits];
    counts_of(sh, counts);
    find_digit(sh, counts, rank);
    prefix |= sh.found[0] << kShift[pass];
    mask = ~0u << kShift[pass];
    rank = sh.found[1];
  }
  // of the list's part before this group: above and equal
  const uint32_t part = sh.found[4];
  uint32_t na = 0, ne = 0;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < part; i += kThreads) {
    const uint32_t k = g.list[i];
    na += k > prefix ? 1u : 0u, ne += k == prefix ? 1u : 0u;
  }
  na = wave_scan(na), ne = wave_scan(ne);
  __syncthreads();  // (`part` is read)
  if (threadIdx.x == 0) sh.found[4] = 0;
  __syncthreads();
  if (lane == 63) {
    if (na != 0) atomicAdd(&sh.found[3], na);
    if (ne != 0) atomicAdd(&sh.found[4], ne);
  }
  __syncthreads();
  uint32_t above = sh.found[3], equal = sh.found[4];
  for (int base = g.first; base < g.end; base += kSpan) {
    if (base > g.first) c.load(base, held);
    write_indices(sh, held, base, prefix, rank, c.index, above, equal);
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

// Workgroups that share a (sequence, kv-head), and how many keys each takes.
static int evict_groups(int nk, int* len) {
  const int spans = (nk - 1) / kSpan + 1, groups = spans < kMaxGroups ? spans : kMaxGroups;
  *len = (spans + groups - 1) / groups * kSpan;  // <= 2^30 / 16 + kSpan
  return (nk - 1) / *len + 1;
}

size_t evict_workspace_bytes(const fa_evict_params& p) {
  if (p.seqlen <= kSpan) return 0;
  int len;
  const size_t groups = (size_t)evict_groups(p.seqlen, &len);
  return (size_t)p.batch * p.heads * (groups * kBins + (size_t)p.seqlen) * sizeof(uint32_t);
}

fa_status run_evict(const fa_evict_params& p, void* workspace, hipStream_t stream, const char** err) {
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
  if (p.seqlen <= kSpan) {
    hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)bh), dim3(kThreads), 0, stream, a);
  } else {
    a.groups = evict_groups(p.seqlen, &a.group_len);
    a.counts = (uint32_t*)workspace;
    a.list = a.counts + bh * a.groups * kBins;
    if (bh * a.groups > INT32_MAX) {
      *err = "grid too large";
      return FA_ERR_UNSUPPORTED;
    }
    for (auto kernel : {evict_count_kernel, evict_list_kernel, evict_index_kernel}) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)(bh * a.groups)), dim3(kThreads), 0, stream, a);
      if (const hipError_t e = hipGetLastError(); e != hipSuccess) return hip_status(e, err);
    }
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.chunks == 0) return hip_status(e, err);
  hipLaunchKernelGGL(gather_rows_kernel, dim3((unsigned)(bh * a.chunks), (unsigned)p.num_tensors + 1), dim3(256), 0, stream,
                     a);
  return hip_status(hipGetLastError(), err);
}

}  // namespace fa
