/*
 * fused_attn_hip.h — C ABI of the MI355X (gfx950) fused-attention backend.
 *
 * This is the drop-in boundary that replaces the reference's pybind module
 * `fused_attn._C` (csrc/bindings.cpp:90-96) and its params struct
 * (csrc/flash_attn.h:9-22), plus the Triton entry points that the reference
 * reached from Python (fused_attn/triton_fwd.py:225-309,
 * fused_attn/triton_splitk.py:140-181, fused_attn/fp8.py:125-147).
 *
 * Conventions
 *  - Plain pointers, element strides and sizes; no framework types.
 *  - All tensor pointers are device pointers on the current HIP device.
 *  - The caller allocates every buffer (outputs and split-K workspace).  The
 *    library never allocates device memory and keeps no pointer after return.
 *  - Every entry point returns an fa_status.  On failure fa_last_error()
 *    returns a thread-local message.  Nothing throws across this boundary and
 *    nothing aborts.
 *  - Work is enqueued on `stream` and is asynchronous, like the reference's
 *    launches on the current CUDA stream (csrc/bindings.cpp:58,78).
 */
#ifndef FUSED_ATTN_HIP_H_
#define FUSED_ATTN_HIP_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Raised by changes that an older caller or library does not survive; added functions keep it
   (fa_attention_fwd_ws and its size query came within 6, and so did the functions of the 4-bit cache and of
   eviction: look them up before use). */
#define FA_ABI_VERSION 6

/* Element types (reference: DType, csrc/flash_attn.h:7). */
typedef enum fa_dtype {
  FA_DTYPE_F16 = 0,
  FA_DTYPE_BF16 = 1,
  FA_DTYPE_F32 = 2,
  FA_DTYPE_FP8_E4M3 = 3, /* OCP float8_e4m3fn, K/V cache only */
  FA_DTYPE_INT4 = 4      /* 4-bit codes, two a byte, with an fp16 (scale, zero) pair a row: fa_cache_params only */
} fa_dtype;

typedef enum fa_status {
  FA_OK = 0,
  FA_ERR_INVALID_ARGUMENT = 1, /* shape / stride / alignment / pointer precondition violated */
  FA_ERR_UNSUPPORTED = 2,      /* valid request this backend does not implement (dtype, head_dim) */
  FA_ERR_WORKSPACE = 3,        /* split-K workspace missing or too small */
  FA_ERR_HIP = 4               /* a HIP runtime call or kernel launch failed */
} fa_status;

/*
 * Forward parameters.  Mirrors AttnParams (csrc/flash_attn.h:9-22) with the
 * varlen, LSE and FP8 fields the Triton paths carried as kernel arguments.
 *
 * Dense layout:  q [B, Hq, Nq, D], k/v [B, Hkv, Nk, D], o like q, any strides
 *                with unit stride along D (strides are in elements); k/v token
 *                strides below 16 MiB.
 * Varlen layout: q [total_q, Hq, D], k/v [total_k, Hkv, D]; `batch` is the
 *                number of sequences, cu_seqlens_q/k are device int32 arrays
 *                of batch+1 prefix offsets starting at 0, the *_stride_b
 *                fields are ignored and *_stride_n is the token stride.
 * Head mapping:  q-head h reads kv-head h / (Hq / Hkv) (reference.py:16-21).
 * Causal:        bottom-right aligned, key j visible to query i iff
 *                j <= i + (Nk - Nq) (reference.py:24-33); a row with no
 *                visible key is written as zeros (reference.py:60-61).
 */
typedef struct fa_fwd_params {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  int64_t q_stride_b, q_stride_h, q_stride_n;
  int64_t k_stride_b, k_stride_h, k_stride_n;
  int64_t v_stride_b, v_stride_h, v_stride_n;
  int64_t o_stride_b, o_stride_h, o_stride_n;
  int32_t batch, heads_q, heads_kv, seqlen_q, seqlen_k, head_dim;
  float scale;   /* softmax scale; callers pass 1/sqrt(D) for the default (ops.py:89) */
  int32_t causal;
  int32_t dtype;    /* fa_dtype of q and o */
  int32_t kv_dtype; /* fa_dtype of k and v: equal to dtype, or FA_DTYPE_FP8_E4M3 */
  /* varlen (NULL for dense) */
  const int32_t* cu_seqlens_q;
  const int32_t* cu_seqlens_k;
  int32_t max_seqlen_q, max_seqlen_k;
  /* optional natural-log LSE output, fp32 (NULL = not written); reference: WRITE_LSE in
     fused_attn/triton_fwd.py:169-172.  Dense: [B, Hq, Nq] at b*lse_stride_b + h*lse_stride_h + n.
     Varlen: [Hq, total_q] at h*lse_stride_h + token (lse_stride_b unused).  Split-K and paged
     decode write it from the combine, dense layout.  A row without keys gets -inf. */
  float* lse;
  int64_t lse_stride_b, lse_stride_h;
  /* FP8 K/V block scales, fp32 [B, Hkv, ceil(Nk/64)] (fused_attn/fp8.py:31-45);
     used only when kv_dtype == FA_DTYPE_FP8_E4M3 */
  const float* k_scale;
  const float* v_scale;
  int64_t scale_stride_b, scale_stride_h;
} fa_fwd_params;

/* Dense FA2 forward.  Replaces attention_fwd_mma (csrc/bindings.cpp:63-81),
   run_attention_fwd_mma (csrc/flash_attn.h:27), attention_fwd (the SIMT kernel,
   csrc/flash_attn.cu:222-228) and attention_triton (fused_attn/triton_fwd.py:225-265).
   f16/bf16 run on the 16-bit MFMA kernel; f32 on the fp32 MFMA at D in {32, 64, 128, 256} and
   on the generic fp32-math kernel at D = 16.  D in {16, 32, 64, 128, 256}. */
fa_status fa_attention_fwd(const fa_fwd_params* p, void* stream);

/* Bytes of workspace fa_attention_fwd_ws wants for these parameters: 0 for a grid that fills the GPU
   by itself, else room for the fp32 partials of the key splits it is cut into (o, (max, sum)).
   Also 0 for parameters that the call would refuse: fa_last_error() is then not empty. */
size_t fa_attention_fwd_workspace_bytes(const fa_fwd_params* p);

/* fa_attention_fwd with a caller workspace of at least fa_attention_fwd_workspace_bytes (16-byte
   aligned; may be NULL when that is 0).  Few queries against many keys leave most compute units
   idle; the key range is then cut over workgroups and a second kernel merges the partials. */
fa_status fa_attention_fwd_ws(const fa_fwd_params* p, void* workspace, size_t workspace_bytes, void* stream);

/* Packed variable-length forward.  Replaces attention_varlen_triton
   (fused_attn/triton_fwd.py:268-309).  Needs cu_seqlens_q/k and max_seqlen_q; optional LSE. */
fa_status fa_attention_varlen_fwd(const fa_fwd_params* p, void* stream);

/* Bytes of workspace fa_attention_splitk needs for `num_splits` key partitions:
   fp32 partial outputs (B*Hq*Nq*S*D floats), each normalised by its own row sum, plus fp32
   (max, sum) pairs (B*Hq*Nq*S*2 floats) in the log2 domain (the reference keeps fp32
   partials too: fused_attn/triton_splitk.py:90-96,156-158).  The library lays them out as
   [B, Hq, Nq, S, D] or, for 32 or more partitions at D <= 128, as [B, Hkv, S, G*Nq, D]
   (G = Hq/Hkv), so that each workgroup's partials are one contiguous block; the layout is
   internal to the split and combine kernels. */
size_t fa_splitk_workspace_bytes(int32_t batch, int32_t heads_q, int32_t seqlen_q, int32_t head_dim,
                                 int32_t num_splits);

/* Split-K flash-decoding: one pass per `split_len`-key partition writing normalised fp32
   partials and fp32 log2-domain statistics, then a log-sum-exp combine kernel (which also
   writes the optional LSE).  f16/bf16 q, D in {64, 128, 256}.  Replaces attention_splitk_triton
   (fused_attn/triton_splitk.py:140-181) and, with kv_dtype == FA_DTYPE_FP8_E4M3 and
   k_scale/v_scale set, attention_fp8_triton (fused_attn/fp8.py:125-147).  split_len must be a
   positive multiple of 64; num_splits = ceil(seqlen_k / split_len). */
fa_status fa_attention_splitk(const fa_fwd_params* p, int32_t split_len, void* workspace,
                              size_t workspace_bytes, void* stream);

/* fa_attention_splitk without a caller workspace, for callers that cannot allocate device memory
   (code under HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).  No
   counterpart in the reference.  Same arguments, validation, kernels and results as
   fa_attention_splitk; the workspace is a static device array the library holds on each GPU for
   the life of the process (FA_SPLITK_NOALLOC_MAX_BYTES), so a request whose
   fa_splitk_workspace_bytes exceeds that size fails with FA_ERR_WORKSPACE.  The library calls no
   allocation routine on this path.  Every call on a GPU uses that GPU's one array: calls that
   overlap on one GPU (other streams, other threads) race and must be serialised by the caller.
   No state in the array has to start at zero (each call writes every partial it reads). */
#define FA_SPLITK_NOALLOC_MAX_BYTES ((size_t)64 << 20)
fa_status fa_attention_splitk_noalloc(const fa_fwd_params* p, int32_t split_len, void* stream);

#define FA_MAX_PAGE_SIZE (1 << 24) /* largest page_size fa_attention_paged_decode accepts */

/* Paged (block-table) K/V for fa_attention_paged_decode.  The K and V pools hold
   num_pages pages of page_size keys; p->k / p->v point at the pools and
   p->k_stride_h / k_stride_n (v likewise) are the head and key strides inside a
   page (p->k_stride_b is unused).  Sequence b's key n lives in page
   block_table[b * block_table_stride + n / page_size] at offset n % page_size. */
typedef struct fa_paged_kv {
  const int32_t* block_table;  /* [batch, block_table_cols] page indices, on the device */
  int64_t block_table_stride;  /* elements between rows of block_table */
  int32_t block_table_cols;    /* pages per sequence in the table; cols * page_size >= p->seqlen_k */
  int32_t page_size;           /* keys per page: a positive multiple of 16 (64 for FP8 pools), at most
                                  FA_MAX_PAGE_SIZE */
  const int32_t* seqlens_k;    /* [batch] keys per sequence, on the device; values above p->seqlen_k
                                  are read as p->seqlen_k, negative values as 0 */
  int32_t num_pages;           /* pages per pool; a table entry outside [0, num_pages) reads as zero keys */
  int32_t reserved;
  int64_t k_page_stride, v_page_stride;  /* elements between consecutive pages of each pool */
} fa_paged_kv;

/* Split-K decode over a paged K/V cache: fa_attention_splitk's kernels (same partials,
   combine, workspace size and split_len rules) with each sequence's keys gathered
   through its block table and its own length seqlens_k[b]; p->seqlen_k is the largest
   length (it sizes the grid) and the causal mask is bottom-right per sequence.
   f16/bf16 q, D in {64, 128, 256}.  The reference lists paged K/V for its decode kernels as a
   roadmap item (README.md:224); the semantics are those of attention_splitk_triton
   (fused_attn/triton_splitk.py:140-181) applied to each sequence's gathered keys.
   FP8 pools (p->kv_dtype == FA_DTYPE_FP8_E4M3): the semantics of attention_fp8_triton
   (fused_attn/fp8.py:125-147) on each sequence's gathered keys.  page_size must then be a
   multiple of 64 and p->k_scale / p->v_scale point at fp32 scale pools
   [num_pages, Hkv, page_size / 64] (the 64-key block scales of each page, as
   fused_attn/fp8.py:31-45 computes them for a [num_pages, Hkv, page_size, D] pool), with
   p->scale_stride_b the elements between pages and p->scale_stride_h between heads; the
   blocks of a page are contiguous.  A page outside [0, num_pages) reads as zero keys. */
fa_status fa_attention_paged_decode(const fa_fwd_params* p, const fa_paged_kv* kv, int32_t split_len,
                                    void* workspace, size_t workspace_bytes, void* stream);

/* Reference split heuristic (fused_attn/triton_splitk.py:130-137):
   min(2*num_cus / (batch*heads), seqlen_k / 256, 64), 1 for seqlen_q > 64. */
int32_t fa_choose_num_splits(int32_t batch, int32_t heads, int32_t seqlen_k, int32_t seqlen_q, int32_t num_cus);

/* 1 when `device` is a gfx950 GPU this library has kernels for, else 0.
   Replaces has_tensor_core_kernel (csrc/bindings.cpp:83-86). */
int32_t fa_device_supported(int32_t device);

/* Thread-local description of the last failure on this thread ("" if none). */
const char* fa_last_error(void);

/* FP8 KV-cache quantiser input: x [batch, heads, seqlen, head_dim] in f32/f16/bf16 with element
   strides (unit head_dim stride); outputs x8 contiguous e4m3fn bytes [batch, heads, seqlen, head_dim]
   and fp32 scales [batch, heads, ceil(seqlen/64)]. */
typedef struct fa_quant_params {
  const void* x;
  int64_t x_stride_b, x_stride_h, x_stride_n;
  int32_t batch, heads, seqlen, head_dim;
  int32_t dtype; /* fa_dtype of x: F16, BF16 or F32 */
  void* x8;
  float* scale;
} fa_quant_params;

/* Per-(batch, head, 64-key block) absmax/448 scaling and e4m3fn rounding, bit-identical to the
   reference's torch chain quantize_kv_fp8 (fused_attn/fp8.py:31-45).  head_dim in {16, 32, 64, 128, 256}. */
fa_status fa_quantize_kv_fp8(const fa_quant_params* p, void* stream);

/*
 * 4-bit K/V cache.  A row (one token of one kv-head, x[D]) is held as D codes of 4 bits and a (scale, zero) pair of
 * fp16:
 *   zero = fp16(lo), scale = fp16((hi - lo) * fp32(1/15))   lo, hi: the row's minimum and maximum, held to +-65504
 *   code = clamp(rint((x - zero) / scale), 0, 15)           fp32, halves to even; 0 where scale is 0
 *   value = code * scale + zero
 * Two codes a byte, channel 2i in the low half of byte i, a row in D/2 contiguous bytes; the pair is one 4-byte word,
 * scale first.  A NaN in a row makes its scale and zero NaN; infinities count as the row's ends.  The reference has no
 * 4-bit cache.
 */
typedef struct fa_int4_params {
  void* x; /* [batch, heads, seqlen, head_dim] F32/F16/BF16, unit head_dim stride, 16-byte aligned with 16-byte strides */
  int64_t x_stride_b, x_stride_h, x_stride_n; /* elements */
  int32_t batch, heads, seqlen, head_dim;     /* head_dim in {64, 128, 256} */
  int32_t dtype;                              /* fa_dtype of x */
  int32_t reserved;
  void* codes; /* rows of head_dim / 2 bytes, 4-byte aligned with strides of whole 4-byte words */
  int64_t codes_stride_b, codes_stride_h, codes_stride_n; /* bytes */
  void* scale; /* (scale, zero) words, 4-byte aligned */
  int64_t scale_stride_b, scale_stride_h, scale_stride_n; /* words */
} fa_int4_params;

/* x -> codes and pairs. */
fa_status fa_quantize_kv_int4(const fa_int4_params* p, void* stream);
/* codes and pairs -> x (rounded once to fp32, once to x's type). */
fa_status fa_dequantize_kv_int4(const fa_int4_params* p, void* stream);

/* New tokens into a cache in place, K and V in one launch: token i of sequence b is written at position
   seqlens_k[b] + i.  k.x / v.x: [batch, heads, new tokens, head_dim], of the same sizes and type; k.codes, k.scale (v
   likewise): the cache, whose stride_b is the one between sequences, or with a block table between pages.  A token
   whose position is outside [0, capacity) (paged: [0, block_table_cols * page_size)), or whose page is outside
   [0, num_pages), is not written. */
typedef struct fa_int4_append_params {
  fa_int4_params k, v;
  const int32_t* seqlens_k; /* [batch], on the device: keys in the cache before the call */
  int64_t capacity;         /* dense: keys a sequence has room for */
  const int32_t* block_table; /* [batch, block_table_cols] or NULL for a dense cache */
  int64_t block_table_stride;
  int32_t block_table_cols, page_size, num_pages, reserved;
} fa_int4_append_params;
fa_status fa_append_kv_int4(const fa_int4_append_params* p, void* stream);

/* Attention over a 4-bit cache (dense or paged), and attention that scores the keys of a dense 4-bit or 16-bit cache:
   fa_attention_splitk's partitions, workspace rule and combine.  f16/bf16 q, head_dim in {64, 128, 256}, bottom-right
   causal mask per sequence; rows without a visible key are zeros. */
typedef struct fa_cache_params {
  const void* q;
  const void* k; /* [batch, heads_kv, seqlen_k, head_dim] in q's type, or codes; paged: pools of pages */
  const void* v;
  void* o;
  int64_t q_stride_b, q_stride_h, q_stride_n;
  int64_t k_stride_b, k_stride_h, k_stride_n; /* elements (codes: bytes), multiples of 16 bytes; paged: stride_b is */
  int64_t v_stride_b, v_stride_h, v_stride_n; /* the page stride, stride_n the one inside a page */
  int64_t o_stride_b, o_stride_h, o_stride_n;
  int32_t batch, heads_q, heads_kv, seqlen_q, seqlen_k, head_dim;
  float scale; /* of at most 1e30 in size */
  int32_t causal;
  int32_t dtype;       /* of q and o */
  int32_t kv_dtype;    /* FA_DTYPE_INT4, or dtype (then scores_out is needed) */
  const void* k_scale; /* 4-bit: the pairs of K and V, 4-byte words; stride_n below 2^22 words */
  const void* v_scale;
  int64_t k_scale_stride_b, k_scale_stride_h, k_scale_stride_n;
  int64_t v_scale_stride_b, v_scale_stride_h, v_scale_stride_n;
  const int32_t* seqlens_k; /* [batch] keys per sequence, on the device, or NULL for seqlen_k each; values above
                               seqlen_k are read as seqlen_k, negative ones as 0.  Rows past them are not read. */
  const int32_t* block_table; /* paged (4-bit only, needs seqlens_k), or NULL; rules as fa_paged_kv */
  int64_t block_table_stride;
  int32_t block_table_cols, page_size, num_pages, reserved;
  float* lse; /* optional natural-log LSE [batch, heads_q, seqlen_q] */
  int64_t lse_stride_b, lse_stride_h;
  /* optional scores, fp32 [batch, heads_kv, seqlen_k] with unit key stride:
       scores_out[b, h, j] = scores_in[b, h, j] + the sum of key j's attention weights over the heads_q / heads_kv
       q-heads and the seqlen_q queries
     (scores_in may be NULL for zeros, or scores_out itself).  Dense caches, and at most 2^23 rows (q-heads x queries)
     a kv-head. */
  const float* scores_in;
  int64_t scores_in_stride_b, scores_in_stride_h;
  float* scores_out;
  int64_t scores_out_stride_b, scores_out_stride_h;
} fa_cache_params;

/* Bytes of workspace fa_attention_cache needs: fa_splitk_workspace_bytes, and with scores 4 bytes for every (q-head,
   query, key), keys rounded up to 32, and 4 for every (q-head, query).  0 for parameters that the call would refuse (a
   split_len that spans more than 258 pages among them), and without a batch or queries. */
size_t fa_attention_cache_workspace_bytes(const fa_cache_params* p, int32_t split_len);
/* split_len: keys a partition, a positive multiple of 64; workspace 16-byte aligned. */
fa_status fa_attention_cache(const fa_cache_params* p, int32_t split_len, void* workspace, size_t workspace_bytes,
                             void* stream);

/* Eviction.  Per (sequence, head) with n = seqlens_k[b] keys: all keys if n <= keep, else the last `recent` ones and the
   keep - recent others of the highest scores (equal scores: the lower index; NaN above every number), in their order.
   index gets their positions (-1 past them), scores_out their scores (0 past them), seqlens_out min(n, keep); row i of
   dst gets row index[i] of src, for every tensor (zero bytes where it is -1). */
#define FA_MAX_EVICT_TENSORS 8
typedef struct fa_evict_tensor {
  const void* src; /* [batch, heads, seqlen] rows of row_bytes contiguous bytes */
  void* dst;       /* [batch, heads, keep] rows; must not overlap any src */
  int64_t src_stride_b, src_stride_h, src_stride_n; /* bytes */
  int64_t dst_stride_b, dst_stride_h, dst_stride_n;
  int64_t row_bytes;
} fa_evict_tensor;
typedef struct fa_evict_params {
  const float* scores; /* [batch, heads, seqlen], unit key stride */
  int64_t scores_stride_b, scores_stride_h;
  const int32_t* seqlens_k; /* [batch] on the device, or NULL for seqlen each; clamped to [0, seqlen] */
  int32_t batch, heads, seqlen, keep, recent; /* 0 <= recent <= keep <= seqlen */
  int32_t num_tensors;
  int32_t* index;       /* [batch, heads, keep] */
  float* scores_out;    /* [batch, heads, keep] */
  int32_t* seqlens_out; /* [batch] */
  fa_evict_tensor tensors[FA_MAX_EVICT_TENSORS];
} fa_evict_params;
/* Bytes of workspace fa_evict_kv needs (16-byte aligned): 0 up to 8192 keys. */
size_t fa_evict_kv_workspace_bytes(const fa_evict_params* p);
fa_status fa_evict_kv(const fa_evict_params* p, void* workspace, size_t workspace_bytes, void* stream);

/* FA_ABI_VERSION of the loaded library. */
int32_t fa_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* FUSED_ATTN_HIP_H_ */
