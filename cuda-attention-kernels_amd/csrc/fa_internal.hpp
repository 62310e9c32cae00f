// Internal interface between the C ABI (fa_abi.cpp) and the kernel launchers
// (fa_prefill.hip, fa_splitk.hip).  Not part of the public header.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/fused_attn_hip.h"

namespace fa {

// Kernel arguments of the prefill and split-K kernels, passed by value.  Pointers are raw
// device pointers; strides are in elements of the pointed-to type.
struct TileArgs {
  const void* q;
  const void* k;
  const void* v;
  void* o;     // prefill: output in the q dtype; split-K: fp32 partials (layout: part_major)
  float* ml;   // split-K: (max, sum) pairs, laid out like the partials
  float* lse;  // prefill: optional natural-log LSE
  const float* k_scale;
  const float* v_scale;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int64_t sqb, sqh, sqn, skb, skh, skn, svb, svh, svn, sob, soh, son;
  int64_t slb, slh;
  int64_t ssb, ssh;
  int32_t hq, hkv, group;
  int32_t nq, nk;  // dense lengths; varlen: maxima
  int32_t n_rowblk;
  int32_t n_split, split_len;
  int32_t ppw, n_chunk;  // split-K: partitions per workgroup, workgroups per (b, kv-head, row block)
  int32_t total;  // workgroups in the grid
  int32_t kv_groups;  // prefill: (batch, kv-head) pairs
  float qk_scale; // softmax scale * log2(e)
  int32_t causal;
  int32_t varlen;
  // paged K/V (split-K decode): k/v are the page pools, skh/skn (svh/svn) strides inside a page
  const int32_t* block_table;
  const int32_t* seqlens_k;
  int64_t sbt;       // block_table row stride
  int64_t spk, spv;  // page strides of the K and V pools
  int32_t page_size, num_pages;
  // key n -> page slot n / page_size as ((uint64_t)n * page_magic) >> page_magic_shift (exact for
  // n < 2^31: page_magic = ceil(2^page_magic_shift / page_size), page_magic_shift = 31 +
  // ceil(log2(page_size)))
  uint32_t page_magic;
  int32_t page_magic_shift;
  // split-K partial layout: 0 = [B, Hq, Nq, S, D] (row-major), 1 = [B, Hkv, S, G*Nq, D]
  // (partition-major: the rows one workgroup writes for one partition are one block)
  int32_t part_major;
  int32_t o16;  // prefill: O base and strides allow 16-byte stores
  // dense prefill: pair heavy and light workgroups on a CU; deal the workgroups to the XCDs
  int32_t fold, deal;
  int32_t share;  // dense causal prefill: q-heads of one XCD, 0 for one order over all heads
  int32_t batch, n_items;  // paged split-K: sequences, and batch * hkv * n_chunk
  int32_t u_heads, u_items;  // dense prefill schedule: q-heads per scheduling unit, and times n_rowblk
};

struct QuantArgs {
  const void* x;
  uint8_t* x8;
  float* scale;
  int64_t sxb, sxh, sxn;
  int32_t h, n, nblk, total;
};

struct CombineArgs {
  const float* opart;  // normalised fp32 partials
  const float* ml;
  void* o;
  int64_t sob, soh, son;
  float* lse;  // optional natural-log LSE [B, Hq, Nq]
  int64_t slb, slh;
  int32_t hq, nq, n_split;
  int32_t group;       // q-heads per kv-head
  int32_t part_major;  // partial layout, as TileArgs::part_major
  int64_t rows;  // prefill: B * Hq * Nq
  const int32_t* seqlens_k;  // paged: the sequences' lengths (clamped to [0, nk])
  int32_t nk, split_len;
};

// 4-bit rows (fa_int4.hip): floats x, codes (bytes) and (scale, zero) pairs (4-byte words), strides in elements.
struct Int4Args {
  const void* x;
  uint8_t* codes;
  uint32_t* pairs;
  int64_t sxb, sxh, sxn, scb, sch, scn, ssb, ssh, ssn;
  int64_t rows;  // batch * h * n
  int32_t h, n;
  int32_t chunks;  // workgroups per (batch, head)
};

struct AppendArgs {
  Int4Args k, v;  // scb and ssb: between sequences, or between pages
  const int32_t* seqlens_k;
  const int32_t* block_table;  // NULL for a dense cache
  int64_t sbt, capacity;
  int32_t page_size, num_pages;
};

// Attention over a 4-bit cache and scored attention (fa_cache.hip).  Strides in elements of what is pointed to (codes:
// bytes; pairs: 4-byte words); paged: the batch strides of k, v and their pairs are page strides.
struct CacheArgs {
  const void *q, *k, *v, *k_scale, *v_scale;
  float* part;  // normalised fp32 partials [B, Hq, Nq, S, D]
  float* ml;    // their (max, sum)
  float* raw;   // scored: log2-domain scores [B, Hkv, raw_tiles, G * Nq, 32 keys]
  int64_t sqb, sqh, sqn, skb, skh, skn, svb, svh, svn;
  int64_t sksb, sksh, sksn, svsb, svsh, svsn;
  int64_t sbt;
  const int32_t* seqlens_k;
  const int32_t* block_table;
  int32_t batch, hq, hkv, group, nq, nk, raw_tiles;
  int32_t n_rowblk, n_split, split_len, n_items, total;
  int32_t causal, page_size, num_pages, page_magic_shift;
  uint32_t page_magic;
  float qk_scale;
};

struct FinishArgs {
  const float* part;  // partials and their (max, sum), as CacheArgs
  const float* ml;
  void* o;
  float* lse;  // written by the merge (may be NULL), or read where use_lse
  const float* raw;
  const float* in;
  float* out;
  int64_t sob, soh, son, slb, slh, sib, sih, sob_s, soh_s, rows;
  const int32_t* seqlens_k;
  int32_t batch, hq, hkv, group, nq, nk, causal, n_split, split_len, chunks, merge_blocks, use_lse, raw_tiles;
  int32_t wide;  // the scores' rows start at 16 bytes
};

// Eviction (fa_evict.hip): strides of the tensors in bytes.
struct EvictTensor {
  const void* src;
  void* dst;
  int64_t sb, sh, sn, db, dh, dn;
  int32_t unit, units;  // bytes a thread copies, and how many make a row
  int32_t shift;        // log2(units), -1 if units is no power of two
};
struct EvictArgs {
  const float* scores;
  int64_t ssb, ssh;
  const int32_t* seqlens_k;
  int32_t* index;
  int32_t* seqlens_out;
  int32_t h, nk, keep, recent, chunks;
  int32_t groups, group_len;  // long caches: workgroups of a (sequence, kv-head), keys of each
  uint32_t *counts, *list;    // and their workspace
  EvictTensor tensors[FA_MAX_EVICT_TENSORS + 1];  // the scores first
};

// Pages (fa_pages.hip): fa_pages_params as the kernels read it.
struct PagesArgs {
  int32_t* block_table;
  int64_t sbt;
  const int32_t *seqlens, *new_lens, *keep_lens;
  const uint8_t* done;
  int32_t* free_pages;
  const int32_t* num_free;
  int64_t* slots;
  int32_t *cu_seqlens, *seqlens_out, *num_free_out;
  int32_t batch, cols, page_size, free_capacity, num_tokens;
  uint32_t capacity;  // keys that a request may hold
};
struct AppendPagedArgs {
  const void *k, *v;
  void *k_cache, *v_cache;
  int64_t skt, skh, svt, svh, skp, skch, skcn, svp, svch, svcn;  // elements
  const int64_t* slots;
  int64_t num_slots;
  int32_t heads, pieces, page_size, total;  // pieces: 16-byte pieces of a row; total: of all rows
};

// Number of rows (q-heads x queries) one split-K workgroup covers, and the
// workgroup shape chosen for a given row count G*Nq.
int splitk_waves_for_rows(int rows);

// TileArgs fields that prefill and split-K share (pointers, strides, heads, scale).
TileArgs common_args(const fa_fwd_params& p);
// and those of paged K/V.
void paged_args(TileArgs& a, const fa_paged_kv& kv);

inline fa_status hip_status(hipError_t e, const char** err) {
  if (e == hipSuccess) return FA_OK;
  if (*err == nullptr) *err = hipGetErrorString(e);  // (a launcher may have said more)
  return FA_ERR_HIP;
}

// Launchers.  They assume fa_abi.cpp has validated `p`.
fa_status run_fwd(const fa_fwd_params& p, bool varlen, hipStream_t stream, const char** err, void* workspace = nullptr);
// Workspace run_fwd wants for a dense call (0: none; without one it runs unsplit).
size_t fwd_workspace_bytes(const fa_fwd_params& p);
// How run_fwd cuts a 16-bit call up: waves (of 32 queries) per workgroup, key splits per row block.
struct FwdPlan {
  int nw, n_split;
  bool short_tile;  // D=64 and D=32: 64-key tiles, three workgroups per CU
};
constexpr int kMaxFwdSplit = 32;
FwdPlan plan_fwd(const fa_fwd_params& p, bool varlen, bool workspace);
// fp32 at head dim 16 (fa_generic.hip); run_fwd forwards it here.
fa_status run_fwd_generic(const fa_fwd_params& p, bool varlen, hipStream_t stream, const char** err);
// fp32 at head dims 32 to 256 on the fp32 MFMA (fa_prefill_f32.hip); run_fwd forwards those here.
fa_status run_fwd_f32(const fa_fwd_params& p, bool varlen, hipStream_t stream, const char** err);
fa_status run_quantize_fp8(const fa_quant_params& p, hipStream_t stream, const char** err);
// Largest workspace the no-allocation split-K entry point holds (a static device array per GPU).
constexpr size_t kSplitkScratchBytes = size_t{64} << 20;
// This device's address of that array (looked up once per device), for fa_attention_splitk_noalloc.
fa_status splitk_scratch(void** ptr, const char** err);
// The merge of split-K partials (fa_splitk.hip) for head dim d and bf16 or fp16 output.
fa_status run_combine(const CombineArgs& c, int d, bool bf16, int64_t rows, hipStream_t stream, const char** err);
// read: floats from codes; else codes from floats
fa_status run_int4_rows(const fa_int4_params& p, bool read, hipStream_t stream, const char** err);
fa_status run_append_int4(const fa_int4_append_params& p, hipStream_t stream, const char** err);
// Why a call of valid parameters cannot be launched, or NULL.
const char* cache_refusal(const fa_cache_params& p, int32_t split_len);
size_t cache_workspace_bytes(const fa_cache_params& p, int32_t split_len);
fa_status run_cache(const fa_cache_params& p, int32_t split_len, void* workspace, hipStream_t stream, const char** err);
size_t evict_workspace_bytes(const fa_evict_params& p);
fa_status run_evict(const fa_evict_params& p, void* workspace, hipStream_t stream, const char** err);
fa_status run_allocate_pages(const fa_pages_params& p, hipStream_t stream, const char** err);
fa_status run_release_pages(const fa_pages_params& p, hipStream_t stream, const char** err);
fa_status run_append_paged(const fa_append_paged_params& p, hipStream_t stream, const char** err);
// kv: paged K/V (nullptr for a dense cache)
fa_status run_splitk(const fa_fwd_params& p, int32_t split_len, void* workspace, hipStream_t stream,
                     const char** err, const fa_paged_kv* kv = nullptr);

// Attention behind shared prefixes (fa_shared.hip): how a call is cut up.
struct SharedPlan {
  int32_t max_prefix, max_suffix;      // bounds of the shared keys, and of a request's keys behind them
  int32_t prefix_split, suffix_split;  // keys per partition
  int32_t prefix_parts, suffix_parts;  // partitions
  int64_t prefix_blocks;               // row blocks of all groups, at most
};
SharedPlan plan_shared(const fa_fwd_params& p, const fa_shared_prefix& s, int page_size);
// Why a call of valid parameters cannot be launched, or NULL.
const char* shared_refusal(const fa_fwd_params& p, const fa_paged_kv& kv, const fa_shared_prefix& s);
size_t shared_workspace_bytes(const fa_fwd_params& p, const fa_paged_kv& kv, const fa_shared_prefix& s);
fa_status run_shared(const fa_fwd_params& p, const fa_paged_kv& kv, const fa_shared_prefix& s, void* workspace,
                     hipStream_t stream, const char** err);

}  // namespace fa
