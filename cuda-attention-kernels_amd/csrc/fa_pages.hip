// Pages of a K/V cache: block tables and slots from request lengths, pages given back, K/V rows written at their slots
// (gfx950).
//
//   have_b = ceil(n_b / page), want_b = ceil((n_b + m_b) / page)   n_b keys held, m_b new tokens
//   need_b = want_b - have_b                                        pages that request b takes
//   first_b = sum of need over the earlier requests                 its place among all pages taken
//   table[b, have_b + j] = free_pages[num_free - 1 - first_b - j]   (the list is taken from its end)
//   slot of packed token t of request b, at position p = n_b + t - begin_b:  table[b, p / page] * page + p % page
//
// Both sums are prefix sums over the batch.  A call is a few hundred to some hundred thousand whole numbers: it is
// bound by its launch and by the chain length load -> two scans -> page load -> store, not by bytes.  So every
// workgroup scans the whole batch for itself, 1024 requests at a time, instead of waiting for another launch's or
// workgroup's sums, and then finds the request of each of its 256 tokens by a binary search in LDS.  A workgroup
// stops scanning behind its last token; the first one writes the per-request outputs.  64 requests of one token 4.2 us,
// 512 with 116000 tokens (454 workgroups) 6.4; giving back 329000 pages of 1024 requests 7.8.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fa_device.hpp"
#include "fa_internal.hpp"

namespace fa {
namespace {

constexpr int kBlock = 256, kPer = 4, kTile = kBlock * kPer;  // threads; requests a thread and a workgroup scan at a time
constexpr uint32_t kLimit = 0x7fffffffu;                      // where sums saturate: above every count that is accepted
constexpr uint32_t kRefused = 0xffffffffu;

// a + b of counts of at most kLimit, held there (an associative sum: the scans may group it as they like).
__device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) { return min(a + b, kLimit); }

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t from_lane(uint32_t x) {  // 0 for lanes that have no source
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
// Inclusive prefix sum over a wave: within rows of 16 lanes, then row ends to the rows behind them.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x = add(x, from_lane<0x111, 0xf>(x));  // row_shr:1
  x = add(x, from_lane<0x112, 0xf>(x));
  x = add(x, from_lane<0x114, 0xf>(x));
  x = add(x, from_lane<0x118, 0xf>(x));
  x = add(x, from_lane<0x142, 0xa>(x));  // row_bcast:15 into rows 1 and 3
  x = add(x, from_lane<0x143, 0xc>(x));  // row_bcast:31 into rows 2 and 3
  return x;
}
// Exclusive prefix sum over the workgroup of one count a thread, on top of `carry`, which becomes the sum of all.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* waves, uint32_t& carry) {
  const uint32_t inc = wave_scan(x);
  const int wave = (int)threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 63) waves[wave] = inc;
  __syncthreads();
  uint32_t before = carry;
#pragma unroll
  for (int w = 0; w < kBlock / 64; ++w) {
    if (w < wave) before = add(before, waves[w]);
    carry = add(carry, waves[w]);
  }
  // (exclusive within the wave: the neighbour's inclusive sum, which saturation makes no difference of)
  const uint32_t left = (uint32_t)__shfl_up((int)inc, 1);
  return add(before, (threadIdx.x & 63) == 0 ? 0u : left);
}

// The first of `count` ascending ends above t.
__device__ __forceinline__ int find(const uint32_t* ends, int count, uint32_t t) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > t) {
      hi = mid;
    } else {
      lo = mid + 1;
    }
  }
  return lo;
}

__device__ __forceinline__ uint32_t pages_of(uint32_t keys, uint32_t page) { return (keys + page - 1) / page; }

}  // namespace

__global__ void __launch_bounds__(kBlock) allocate_pages_kernel(const PagesArgs a) {
  __shared__ uint32_t s_end[kTile], s_held[kTile], s_first[kTile];
  __shared__ uint32_t s_wave[2][kBlock / 64];
  __shared__ uint32_t s_used;
  const uint32_t page = (uint32_t)a.page_size;
  const uint32_t free = (uint32_t)min(max(a.num_free[0], 0), a.free_capacity);
  const uint32_t tokens = (uint32_t)a.num_tokens, t = blockIdx.x * (uint32_t)kBlock + threadIdx.x;
  const bool first_wg = blockIdx.x == 0;
  uint32_t token_sum = 0, page_sum = 0;
  int64_t slot = -1;
  if (threadIdx.x == 0) s_used = 0;
  if (first_wg && threadIdx.x == 0) a.cu_seqlens[0] = 0;
  for (int base = 0; base < a.batch; base += kTile) {
    const int count = min(a.batch - base, kTile), i0 = (int)threadIdx.x * kPer;
    uint32_t n[kPer], m[kPer], sum = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const bool in = i0 + k < count;
      n[k] = in ? (uint32_t)max(a.seqlens[base + i0 + k], 0) : 0u;
      m[k] = in ? (uint32_t)max(a.new_lens[base + i0 + k], 0) : 0u;
      sum = add(sum, m[k]);
    }
    const uint32_t tile_begin = token_sum;
    uint32_t end = block_scan(sum, s_wave[0], token_sum);
    uint32_t need[kPer], pages = 0;
    bool fits[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      end = add(end, m[k]);
      if (i0 + k < count) s_end[i0 + k] = end;
      fits[k] = i0 + k < count && n[k] + m[k] <= a.capacity && end <= tokens;
      need[k] = fits[k] ? pages_of(n[k] + m[k], page) - pages_of(n[k], page) : 0u;
      pages = add(pages, need[k]);
      if (first_wg && i0 + k < count) a.cu_seqlens[base + i0 + k + 1] = (int32_t)min(end, tokens);
    }
    uint32_t taken = block_scan(pages, s_wave[1], page_sum), used = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const uint32_t from = taken;
      taken = add(taken, need[k]);
      const bool ok = fits[k] && (need[k] == 0 || taken <= free);
      if (ok && need[k] > 0) used = taken;
      if (i0 + k < count) {
        s_held[i0 + k] = n[k];
        s_first[i0 + k] = ok ? from : kRefused;
        if (first_wg) a.seqlens_out[base + i0 + k] = (int32_t)(ok ? n[k] + m[k] : n[k]);
      }
    }
    if (first_wg && used > 0) atomicMax(&s_used, used);
    __syncthreads();
    if (t >= tile_begin && t < min(token_sum, tokens)) {
      const int i = find(s_end, count, t);
      const uint32_t first = s_first[i], held = s_held[i];
      if (first != kRefused) {
        const uint32_t pos = held + (t - (i > 0 ? s_end[i - 1] : tile_begin));
        const uint32_t col = pos / page, off = pos - col * page, have = pages_of(held, page);
        int32_t* entry = a.block_table + (int64_t)(base + i) * a.sbt + col;
        int32_t at;
        if (col < have) {
          at = *entry;  // (entries of pages held are written by no thread)
        } else {
          at = a.free_pages[free - 1 - (first + (col - have))];
          if (off == 0) *entry = at;  // a new page's first token
        }
        slot = at >= 0 ? (int64_t)at * page + off : -1;
      }
    }
    // uniform: this workgroup's tokens all lie in the requests scanned so far
    if (!first_wg && token_sum > blockIdx.x * (uint32_t)kBlock + (kBlock - 1)) break;
    __syncthreads();
  }
  if (t < tokens) a.slots[t] = slot;
  if (first_wg && threadIdx.x == 0) {
    if (a.batch == 0) s_used = 0;
    a.num_free_out[0] = (int32_t)(free - s_used);
  }
}

// Pages of finished requests behind those they share, onto the end of the list: in order of requests, then of columns.
__global__ void __launch_bounds__(kBlock) release_pages_kernel(const PagesArgs a) {
  __shared__ uint32_t s_end[kTile], s_from[kTile], s_ok[kTile];
  __shared__ uint32_t s_wave[kBlock / 64];
  __shared__ uint32_t s_given;
  const uint32_t page = (uint32_t)a.page_size, cols = (uint32_t)a.cols;
  const uint32_t free = (uint32_t)min(max(a.num_free[0], 0), a.free_capacity), room = (uint32_t)a.free_capacity - free;
  const bool first_wg = blockIdx.x == 0;
  uint32_t page_sum = 0;
  if (threadIdx.x == 0) s_given = 0;
  for (int base = 0; base < a.batch; base += kTile) {
    const int count = min(a.batch - base, kTile), i0 = (int)threadIdx.x * kPer;
    uint32_t n[kPer], keep[kPer], pages[kPer], sum = 0;
    bool done[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const bool in = i0 + k < count;
      n[k] = in ? (uint32_t)max(a.seqlens[base + i0 + k], 0) : 0u;
      keep[k] = in && a.keep_lens != nullptr ? (uint32_t)max(a.keep_lens[base + i0 + k], 0) / page : 0u;
      done[k] = in && a.done[base + i0 + k] != 0;
      const uint32_t have = min(pages_of(n[k], page), cols);
      pages[k] = done[k] && have > keep[k] ? have - keep[k] : 0u;
      sum = add(sum, pages[k]);
    }
    const uint32_t tile_begin = page_sum;
    uint32_t end = block_scan(sum, s_wave, page_sum), given = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      end = add(end, pages[k]);
      const bool ok = done[k] && (pages[k] == 0 || end <= room);
      if (ok && pages[k] > 0) given = end;
      if (i0 + k < count) {
        s_end[i0 + k] = end;
        s_from[i0 + k] = keep[k];
        s_ok[i0 + k] = ok;
        if (first_wg) a.seqlens_out[base + i0 + k] = (int32_t)(ok ? 0u : n[k]);
      }
    }
    if (first_wg && given > 0) atomicMax(&s_given, given);
    __syncthreads();
    // the pages of this tile, dealt to the workgroups 256 at a time (those past the list's room belong to refused requests)
    const uint32_t tile_end = min(page_sum, room);
    for (uint32_t i = tile_begin + blockIdx.x * (uint32_t)kBlock + threadIdx.x; i < tile_end; i += gridDim.x * (uint32_t)kBlock) {
      const int s = find(s_end, count, i);
      if (s_ok[s]) {
        const uint32_t col = s_from[s] + (i - (s > 0 ? s_end[s - 1] : tile_begin));
        a.free_pages[free + i] = a.block_table[(int64_t)(base + s) * a.sbt + col];
      }
    }
    __syncthreads();
  }
  if (first_wg && threadIdx.x == 0) {
    if (a.batch == 0) s_given = 0;
    a.num_free_out[0] = (int32_t)(free + s_given);
  }
}

// K/V rows of packed tokens to their slots, K and V in one launch: one read and one write of every row.  A thread
// moves kCopy 16-byte pieces of K and of V, whose loads are in flight together with those of the slots.  40001 tokens of 8
// heads x 128, 328 MB: 63.9 us a call on buffers in turn, 5.1 TB/s (two torch copies of the same: 65); 58-59 under the profiler on
// the same buffers, parts of which stay in the caches; 64 tokens 4.2 us.
constexpr int kCopy = 4;

__global__ void __launch_bounds__(kBlock) append_kv_paged_kernel(const AppendPagedArgs a) {
  const uint32_t first = blockIdx.x * (uint32_t)(kBlock * kCopy) + threadIdx.x;
  const uint32_t pieces = (uint32_t)a.pieces;  // of a head's row
  u32x4 k[kCopy], v[kCopy];
  int64_t slot[kCopy];
  uint32_t head[kCopy], piece[kCopy];
#pragma unroll
  for (int u = 0; u < kCopy; ++u) {
    const uint32_t i = first + u * kBlock;
    slot[u] = -1;
    if (i < (uint32_t)a.total) {
      const uint32_t row = i / pieces, token = row / (uint32_t)a.heads;
      head[u] = row - token * (uint32_t)a.heads;
      piece[u] = i - row * pieces;
      slot[u] = a.slots[token];
      k[u] = ld16((const uint16_t*)a.k + token * a.skt + head[u] * a.skh + piece[u] * 8);
      v[u] = ld16((const uint16_t*)a.v + token * a.svt + head[u] * a.svh + piece[u] * 8);
    }
  }
#pragma unroll
  for (int u = 0; u < kCopy; ++u) {
    if (slot[u] < 0 || slot[u] >= a.num_slots) continue;
    const uint32_t s = (uint32_t)slot[u], page = s / (uint32_t)a.page_size, off = s - page * (uint32_t)a.page_size;
    st16((uint16_t*)a.k_cache + page * a.skp + head[u] * a.skch + off * a.skcn + piece[u] * 8, k[u]);
    st16((uint16_t*)a.v_cache + page * a.svp + head[u] * a.svch + off * a.svcn + piece[u] * 8, v[u]);
  }
}

static PagesArgs pages_args(const fa_pages_params& p) {
  PagesArgs a{};
  a.block_table = p.block_table;
  a.sbt = p.block_table_stride;
  a.seqlens = p.seqlens;
  a.new_lens = p.new_lens;
  a.done = p.done;
  a.keep_lens = p.keep_lens;
  a.free_pages = p.free_pages;
  a.num_free = p.num_free;
  a.slots = p.slots;
  a.cu_seqlens = p.cu_seqlens;
  a.seqlens_out = p.seqlens_out;
  a.num_free_out = p.num_free_out;
  a.batch = p.batch;
  a.cols = p.block_table_cols;
  a.page_size = p.page_size;
  a.free_capacity = p.free_capacity;
  a.num_tokens = p.num_tokens;
  a.capacity = (uint32_t)std::min<int64_t>((int64_t)p.block_table_cols * p.page_size, INT32_MAX);
  return a;
}

fa_status run_allocate_pages(const fa_pages_params& p, hipStream_t stream, const char** err) {
  const unsigned grid = (unsigned)std::max<int64_t>(1, ((int64_t)p.num_tokens + kBlock - 1) / kBlock);
  hipLaunchKernelGGL(allocate_pages_kernel, dim3(grid), dim3(kBlock), 0, stream, pages_args(p));
  return hip_status(hipGetLastError(), err);
}

fa_status run_release_pages(const fa_pages_params& p, hipStream_t stream, const char** err) {
  // at most 8 pages of the table a thread, and two workgroups a compute unit
  const int64_t entries = (int64_t)p.batch * p.block_table_cols;
  const unsigned grid = (unsigned)std::min<int64_t>(std::max<int64_t>(1, entries / (kBlock * 8)), 512);
  hipLaunchKernelGGL(release_pages_kernel, dim3(grid), dim3(kBlock), 0, stream, pages_args(p));
  return hip_status(hipGetLastError(), err);
}

fa_status run_append_paged(const fa_append_paged_params& p, hipStream_t stream, const char** err) {
  AppendPagedArgs a{};
  a.k = p.k;
  a.v = p.v;
  a.skt = p.k_stride_t;
  a.skh = p.k_stride_h;
  a.svt = p.v_stride_t;
  a.svh = p.v_stride_h;
  a.k_cache = p.k_cache;
  a.v_cache = p.v_cache;
  a.skp = p.k_page_stride;
  a.skch = p.k_cache_stride_h;
  a.skcn = p.k_cache_stride_n;
  a.svp = p.v_page_stride;
  a.svch = p.v_cache_stride_h;
  a.svcn = p.v_cache_stride_n;
  a.slots = p.slots;
  a.num_slots = (int64_t)p.num_pages * p.page_size;
  a.heads = p.heads;
  a.pieces = p.head_dim / 8;
  a.page_size = p.page_size;
  const int64_t total = (int64_t)p.num_tokens * p.heads * a.pieces;
  if (total > INT32_MAX - kBlock * kCopy) {
    *err = "too many rows";
    return FA_ERR_UNSUPPORTED;
  }
  a.total = (int32_t)total;
  const unsigned grid = (unsigned)((total + kBlock * kCopy - 1) / (kBlock * kCopy));
  hipLaunchKernelGGL(append_kv_paged_kernel, dim3(grid), dim3(kBlock), 0, stream, a);
  return hip_status(hipGetLastError(), err);
}

}  // namespace fa
