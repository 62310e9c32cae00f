// Requests in groups that share the start of their keys: which keys of a request are read once for its group.
//
// The kernels split a group's prefix at a multiple of kPrefixUnit keys: the keys below it (the "shared" ones) are read
// for all rows of the group at once, those from it on through each request's own block-table row.  64 keys are a whole
// tile, a whole FP8 scale block and whole page groups of every page size, so both parts address memory as an unsplit
// sequence would.
#pragma once

#include "fa_device.hpp"
#include "fa_internal.hpp"

namespace fa {

constexpr int kPrefixUnit = 64;
constexpr int kPrefixPages = 128;  // pages that a partition of the shared keys may span,
constexpr int kSuffixPages = 256;  // and one of a request's own
constexpr int kFp8Keys = 64 * 64;  // keys of an FP8 partition: a lane holds a 64-key block's scales

// The V scales of an FP8 partition (lane i: block i) as units in which O can be held: 0 for a block whose values count as 0
// (a scale of 0, or below 2^-90 of the partition's largest, in which O would overflow: O is at most 448 codes x 2^8 (P) x
// 2^12 keys, 2^29), NaN for an infinite one or NaN, whose block makes NaN of every row that sees it.  Every lane calls it.
__device__ __forceinline__ float v_units(float scale) {
  const float size = fabsf(scale);
  const bool finite = size < __builtin_inff();
  float top = finite ? size : 0.f;
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
  return !finite ? __builtin_nanf("") : size > top * 0x1p-90f ? scale : 0.f;
}
// Neither 0 nor NaN, of a uniform value.
__device__ __forceinline__ bool is_unit(float unit) {
  return (__builtin_bit_cast(uint32_t, unit) & 0x7fffffffu) - 1u < 0x7f7fffffu;
}
// The first block without a value among the units of a partition, at most 64 (uniform).
__device__ __forceinline__ int first_without_value(float units) {
  const uint64_t none = __builtin_amdgcn_ballot_w64(units != units);
  return none != 0 ? __builtin_ctzll(none) : 64;
}

// Division of 0 <= n < 2^31 by a number that the host knows: (n * mul) >> shift.
struct FastDiv {
  uint32_t mul;
  int32_t shift;
  __host__ static FastDiv by(int32_t d) {
    int lg = 0;
    while ((int64_t{1} << lg) < (int64_t)d) ++lg;
    return {(uint32_t)(((uint64_t{1} << (31 + lg)) + (uint64_t)d - 1) / (uint64_t)d), 31 + lg};
  }
  __device__ __forceinline__ int of(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
};

struct SharedArgs {
  const int32_t* prefix_lens;  // [groups], or NULL: max_prefix for every group
  const int32_t* cu_groups;    // [groups + 1], or NULL: one group of the whole batch
  int32_t groups, batch;
  int32_t max_prefix, max_suffix;  // bounds of the prefixes, and of a request's keys behind its own
  int32_t table_keys;              // keys that a block-table row can name
  int32_t part_base, part_stride;  // a row's partials: part_stride of them, those of its own keys from part_base on
  int32_t prefix_split, suffix_split;  // keys per partition
  int32_t suffix_blocks;               // blocks of 32 rows of a request
  FastDiv by_page, by_hkv, by_group, by_nq, by_batch, by_prefix_blocks, by_suffix_blocks;
  // the grid: prefix_first workgroups of the shared keys, suffix_wgs of the requests' own, the rest of the shared keys'
  int32_t prefix_first, suffix_wgs;
};

struct SharedTileArgs : TileArgs {
  SharedArgs shared;
};

// The prefix of group g (in range), and how many of its keys are shared.
__device__ __forceinline__ int prefix_of(const SharedArgs& s, int g) {
  return s.prefix_lens != nullptr ? min(max(s.prefix_lens[g], 0), s.max_prefix) : s.max_prefix;
}
__device__ __forceinline__ int shared_keys(const SharedArgs& s, int prefix) {
  return min(prefix, s.table_keys) / kPrefixUnit * kPrefixUnit;
}

// Keys that a request is read to have, behind a prefix of `prefix`.
__device__ __forceinline__ int keys_of(const SharedArgs& s, int seqlen, int prefix) {
  return min(max(seqlen, 0), min(prefix + s.max_suffix, s.table_keys));
}

// Requests [b0, b1) of group g (in range), within the batch whatever cu_groups holds.
__device__ __forceinline__ void group_range(const SharedArgs& s, int g, int& b0, int& b1) {
  b0 = 0;
  b1 = s.batch;
  if (s.cu_groups != nullptr) {
    b0 = min(max(s.cu_groups[g], 0), s.batch);
    b1 = min(max(s.cu_groups[g + 1], b0), s.batch);
  }
}

// The prefix of request b (uniform over the wave; every lane calls it).  A request of no group has none.
__device__ __forceinline__ int prefix_of_request(const SharedArgs& s, int b) {
  if (s.cu_groups == nullptr) return __builtin_amdgcn_readfirstlane(prefix_of(s, 0));
  const int lane = (int)threadIdx.x & 63;
  for (int base = 0; base < s.groups; base += 64) {
    const int g = base + lane;
    int b0 = 0, b1 = 0, keys = 0;
    if (g < s.groups) {
      group_range(s, g, b0, b1);
      keys = prefix_of(s, g);  // (every lane its group's: the loads are in flight together)
    }
    const uint64_t in = __builtin_amdgcn_ballot_w64(b0 <= b && b < b1);
    if (in != 0) return __builtin_amdgcn_readlane(keys, __builtin_ctzll(in));
  }
  return 0;
}

// The requests [b0, b1) and the prefix of the group that row block `rb` belongs to, and the block within it, when a group
// of n requests has ceil(n * rows_each / rows) blocks (uniform; every lane calls it).  False past the last block.
__device__ __forceinline__ bool group_of_block(const SharedArgs& s, int rows_each, int rows, int& rb, int& b0, int& b1, int& prefix) {
  const int lane = (int)threadIdx.x & 63;
  if (s.cu_groups == nullptr) {
    b0 = 0;
    b1 = s.batch;
    prefix = __builtin_amdgcn_readfirstlane(prefix_of(s, 0));
    return rb < (s.batch * rows_each + rows - 1) / rows;
  }
  for (int base = 0; base < s.groups; base += 64) {
    int lo = 0, hi = 0, k = 0;
    if (base + lane < s.groups) {
      group_range(s, base + lane, lo, hi);
      k = prefix_of(s, base + lane);
    }
    const int blocks = ((hi - lo) * rows_each + rows - 1) / rows;
    int end = blocks;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int left = __shfl_up(end, d);
      end += lane >= d ? left : 0;
    }
    const uint64_t in = __builtin_amdgcn_ballot_w64(end > rb);
    if (in != 0) {
      const int at = __builtin_ctzll(in);
      prefix = __builtin_amdgcn_readlane(k, at);
      b0 = __builtin_amdgcn_readlane(lo, at);
      b1 = __builtin_amdgcn_readlane(hi, at);
      rb -= __builtin_amdgcn_readlane(end - blocks, at);
      return true;
    }
    rb -= __builtin_amdgcn_readlane(end, 63);
  }
  return false;
}

// The request of [b0, b1) whose block-table row names the group's shared keys: the first that holds them all, or else the
// first of the longest; `longest`: how many of them it holds (uniform; every lane calls it).
__device__ __forceinline__ int prefix_holder(const int32_t* seqlens, int b0, int b1, int keys, int& longest) {
  const int lane = (int)threadIdx.x & 63;
  int best = b0;
  longest = 0;
  for (int base = b0; base < b1; base += 64) {
    const int n = base + lane < b1 ? min(seqlens[base + lane], keys) : 0;
    const uint64_t whole = __builtin_amdgcn_ballot_w64(n == keys);
    if (whole != 0) {
      longest = keys;
      return base + __builtin_ctzll(whole);
    }
    int top = n;
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) top = max(top, __shfl_xor(top, d));
    top = __builtin_amdgcn_readfirstlane(top);
    if (top > longest) {
      longest = top;
      best = base + __builtin_ctzll(__builtin_amdgcn_ballot_w64(n == top));
    }
  }
  return best;
}

template <class F>
hipError_t by_dim_and_type(int d, bool bf, F&& f) {
  auto type = [&](auto dim) { return bf ? f(dim, BF16{}) : f(dim, F16{}); };
  if (d == 64) return type(std::integral_constant<int, 64>{});
  if (d == 128) return type(std::integral_constant<int, 128>{});
  return type(std::integral_constant<int, 256>{});
}

}  // namespace fa
