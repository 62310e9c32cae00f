// Attention of requests that share the start of their keys (gfx950).
//
// A group's shared keys meet the rows of all its requests (requests x q-heads of a kv-head x queries) as one product: the
// pipelined prefill kernel over pages (attn_fwd_kernel, SHARED), 128 rows a workgroup, the keys cut into partitions.  The
// requests' own keys are read by waves of the same launch (suffix_rows), a partition of one request's each.  Every (row,
// partition) of either part leaves a partial, normalised by its own row sum, with its (max, sum); one kernel merges a row's:
//   m = max_s m_s;  w_s = 2^(m_s - m) l_s;  O = sum_s w_s O_s / sum_s w_s   (0 when the sum is 0)
//
// What bounds it: the shared keys' products (matrix cores and, with as many vector cycles, the exponentials) beside the
// stream of the own keys, and about 8 us of start and end.  64 requests of 4 rows a kv-head (8 of them, D = 128) behind
// 8192 keys, up to 512 of their own: 27 us and the merge's 4.8; 32 of 16 rows behind 16384, up to 2000: 56 and 5.9.  Whole
// calls 30 and 61 us; with the split-K kernels over both parts, one after the other, 70 and 114.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fa_prefill_kernel.hpp"
#include "fa_shared.hpp"

namespace fa {

struct MergeArgs {
  float* part;  // [batch, hq, nq, part_stride] partials, then their (m, l) in ml
  const float* ml;
  void* o;
  float* lse;  // optional natural-log LSE
  int64_t sob, soh, son, slb, slh;
  const int32_t* seqlens;
  int32_t hq, nq, chunks;  // chunks: workgroups a request
  int32_t causal;
  FastDiv by_chunks, by_prefix_split, by_suffix_split;
  SharedArgs shared;
  TileArgs tile;  // for partials that are formed anew
  int32_t fp8;
};

// One value of a row: 16-bit E, or an FP8 code.
template <class E>
__device__ __forceinline__ float value_at(const void* p, int64_t at, bool fp8) {
  if (fp8) return __builtin_amdgcn_cvt_pk_f32_fp8((int)((const uint8_t*)p)[at], false)[0];
  return lo_f32<E>(((const uint16_t*)p)[at]);
}

// A row that sees the first keys of a partition only (its request ends there, or its causal end lies there) shared the
// partition's products with rows that see all of it.  Its weight of a key that it does not see is 0, and 0 times an infinity or
// NaN in that key's V is NaN.  So a partial of such a row that is not finite is formed anew, over the keys that it sees: a dot
// product a thread for 256 keys at a time, then a column of V a thread.  Slow, and only ever done where V holds such values;
// other calls pay a comparison a request, and one load and barrier where a request ends among the shared keys.
//
// The workgroup's rows are r0 to r0 + ROWS - 1 of request b, which has `keys` keys; all threads call it.
template <int D, class E, int ROWS>
__device__ __forceinline__ void renew_partials(int b, int r0, int shared, int keys) {
  // (the arguments through a pointer that the compiler does not know: it would load what is used here at the kernel's
  // entry, and spill: 0.5 to 2 us a call)
  uint64_t address = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
#if defined(__HIP_DEVICE_COMPILE__)
  __asm__ volatile("" : "+s"(address));
  const auto& a = *reinterpret_cast<const MergeArgs __attribute__((address_space(4)))*>(address);
#else
  const MergeArgs& a = *reinterpret_cast<const MergeArgs*>(address);
#endif
  __shared__ float s_p[256];
  __shared__ int64_t s_at[256];  // V's row of a key, in elements; -1: no value
  __shared__ float s_scale[256];
  const auto& t = a.tile;
  const int tid = (int)threadIdx.x, rows = min(ROWS, a.hq * a.nq - r0);
  // the row's keys, and the partition that they end in, if that has more
  auto ends_in = [&](int r, int& limit) {
    limit = t.causal ? keys - a.nq + (r - a.shared.by_nq.of(r) * a.nq) + 1 : keys;
    if (limit <= 0 || limit >= shared) return -1;
    const int s = a.by_prefix_split.of(limit - 1);
    return limit < min((s + 1) * a.shared.prefix_split, shared) ? s : -1;
  };
  auto part_of = [&](int r, int s) { return a.part + (((int64_t)b * a.hq * a.nq + r) * a.shared.part_stride + s) * D; };
  bool spoiled = false;
  for (int i = tid; i < rows * (D / 4); i += 256) {
    int limit;
    const int r = r0 + i / (D / 4), s = ends_in(r, limit);
    if (s < 0) continue;
    const f32x4 v = __builtin_bit_cast(f32x4, ld16(part_of(r, s) + i % (D / 4) * 4));
#pragma unroll
    for (int e = 0; e < 4; ++e) spoiled |= !(fabsf(v[e]) < __builtin_inff());
  }
  if (!__syncthreads_or(spoiled)) return;

  const int32_t* bt = t.block_table + (int64_t)b * t.sbt;
  for (int r = r0; r < r0 + rows; ++r) {
    int limit;
    const int s = ends_in(r, limit);
    if (s < 0) continue;
    float* out = part_of(r, s);
    if (!__syncthreads_or(tid < D && !(fabsf(out[tid % D]) < __builtin_inff()))) continue;
    const int h = a.shared.by_nq.of(r), kvh = a.shared.by_group.of(h);
    const uint16_t* q = (const uint16_t*)t.q + (int64_t)b * t.sqb + (int64_t)h * t.sqh + (int64_t)(r - h * a.nq) * t.sqn;
    const float m = a.ml[(((int64_t)b * a.hq * a.nq + r) * a.shared.part_stride + s) * 2], m_safe = m == -__builtin_inff() ? 0.f : m;
    float acc = 0.f, sum = 0.f;
    for (int n0 = s * a.shared.prefix_split; n0 < limit; n0 += 256) {
      const int n = n0 + tid;
      float p = 0.f;
      s_at[tid] = -1;
      if (n < limit) {
        const int slot = a.shared.by_page.of(n), page = bt[slot], off = n - slot * t.page_size;
        float score = 0.f, c = fabsf(t.qk_scale);
        if ((uint32_t)page < (uint32_t)t.num_pages) {  // (keys outside the pool are zeros)
          const int64_t at = (int64_t)page * t.spk + (int64_t)kvh * t.skh + (int64_t)off * t.skn;
#pragma unroll 4
          for (int d = 0; d < D; ++d) score += lo_f32<E>(q[d]) * value_at<E>(t.k, at + d, a.fp8);
          s_at[tid] = (int64_t)page * t.spv + (int64_t)kvh * t.svh + (int64_t)off * t.svn;
          if (a.fp8) {
            const int64_t block = (int64_t)page * t.ssb + (int64_t)kvh * t.ssh + off / 64;
            const float vs = t.v_scale[block];
            c *= t.k_scale[block];
            s_scale[tid] = fabsf(vs) < __builtin_inff() ? vs : __builtin_nanf("");
            if (vs == 0.f) s_at[tid] = -1;
          }
        } else {
          c = 0.f;
        }
        p = fast_exp2((t.qk_scale < 0.f ? -score : score) * fmaxf(c, kMinScale) - m_safe);
      }
      s_p[tid] = p;
      __syncthreads();
      const int count = min(limit - n0, 256);
      for (int i = 0; i < count; ++i) {
        const float w = s_p[i];
        sum += w;
        if (tid < D && s_at[i] >= 0) acc += w * (value_at<E>(t.v, s_at[i] + tid, a.fp8) * (a.fp8 ? s_scale[i] : 1.f));
      }
      __syncthreads();
    }
    if (tid < D) out[tid] = sum == 0.f ? 0.f : acc / sum;
  }
  __syncthreads();
}

// Bound by its launch, and by the partials' bytes where they are many (2048 rows x 10 partials of D = 128: 4.8 us; a
// workgroup for every row, the partials dealt to its threads, took 8.4; 8192 rows 8.9).  Few instructions a row: with 8
// partials a thread in place of 4, most of them none, and divisions by numbers that the host knows, the latter took 11.
//
// A thread merges 4 values of a row over every WAYS-th of its partials, CH of them in flight together; WAYS threads meet
// in LDS.  A workgroup's rows are one request's, so that its group and its partitions are found once, uniformly.
template <int D, class E, int WAYS>
__global__ void __launch_bounds__(256) shared_merge_kernel(const MergeArgs a) {
  constexpr int TPR = D / 4, ROWS = 256 / (TPR * WAYS), CH = WAYS > 1 ? 4 : 8;
  static_assert(ROWS >= 1, "a row per workgroup at least");
  constexpr float NEG_INF = -__builtin_inff();
  __shared__ f32x4 s_acc[WAYS > 1 ? 256 : 1];
  __shared__ f32x2 s_ml[WAYS > 1 ? ROWS * WAYS : 1];
  const int b = a.by_chunks.of((int)blockIdx.x), chunk = (int)blockIdx.x - b * a.chunks;
  const int tid = (int)threadIdx.x, dq = tid % TPR, way = tid / TPR % WAYS, sub = tid / (TPR * WAYS);
  const int rows = a.hq * a.nq, r = chunk * ROWS + sub;  // (q-head, query) of the request
  const int prefix = prefix_of_request(a.shared, b), shared = shared_keys(a.shared, prefix);
  const int keys = keys_of(a.shared, __builtin_amdgcn_readfirstlane(a.seqlens[b]), prefix);
  const int first = a.by_prefix_split.of(shared + a.shared.prefix_split - 1);
  const int count = r < rows ? first + (keys > shared ? a.by_suffix_split.of(keys - shared + a.shared.suffix_split - 1) : 0) : 0;
  const int skip = a.shared.part_base - first;  // places between the two runs of a row's partials
  if ((a.causal ? keys - a.nq + 1 : keys) < shared) renew_partials<D, E, ROWS>(b, chunk * ROWS, shared, keys);  // uniform
  const int64_t base = ((int64_t)b * rows + min(r, rows - 1)) * a.shared.part_stride;
  const float* ml = a.ml + base * 2;
  const float* op = a.part + base * D + 4 * dq;
  float m = NEG_INF, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = way; s0 < count; s0 += CH * WAYS) {
    f32x2 st[CH];
    f32x4 pv[CH];
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      int s = s0 + u * WAYS;
      st[u] = f32x2{NEG_INF, 0.f};
      pv[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (s < count) {
        s += s >= first ? skip : 0;
        st[u] = __builtin_bit_cast(f32x2, ld8(ml + 2 * s));
        pv[u] = __builtin_bit_cast(f32x4, ld16(op + (int64_t)s * D));
      }
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < CH; ++u) mn = fmaxf(mn, st[u][0]);
    const float m_ref = (mn == NEG_INF) ? 0.f : mn;
    const float alpha = fast_exp2(m - m_ref);  // 0 while m = -inf
    l *= alpha;
    acc *= alpha;
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      const float w = fast_exp2(st[u][0] - m_ref) * st[u][1];
      l += w;
      acc += w * pv[u];
    }
    m = mn;
  }
  if constexpr (WAYS > 1) {
    s_acc[tid] = acc;
    if (dq == 0) s_ml[sub * WAYS + way] = f32x2{m, l};
    __syncthreads();
    if (way > 0) return;
    float mn = NEG_INF;
#pragma unroll
    for (int w = 0; w < WAYS; ++w) mn = fmaxf(mn, s_ml[sub * WAYS + w][0]);
    const float m_ref = (mn == NEG_INF) ? 0.f : mn;
    m = mn;
    l = 0.f;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAYS; ++w) {
      const float f = fast_exp2(s_ml[sub * WAYS + w][0] - m_ref);
      l += f * s_ml[sub * WAYS + w][1];
      acc += f * s_acc[(sub * WAYS + w) * TPR + dq];
    }
  }
  if (r >= rows) return;
  const float l_safe = (l == 0.f) ? 1.f : l, inv = 1.f / l_safe;
  const int h = a.shared.by_nq.of(r), n = r - h * a.nq;
  if (a.lse != nullptr && dq == 0) a.lse[b * a.slb + (int64_t)h * a.slh + n] = (m + __log2f(l_safe)) * kLn2;
  uint16_t* o = (uint16_t*)a.o + b * a.sob + (int64_t)h * a.soh + (int64_t)n * a.son + 4 * dq;
  st8(o, u32x2{pack2<E>(acc[0] * inv, acc[1] * inv), pack2<E>(acc[2] * inv, acc[3] * inv)});
}

// ------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------

namespace {

constexpr int kCus = 256;
constexpr int prefix_tile_keys(int d) { return d == 256 ? 32 : 64; }

template <int D, class E>
hipError_t launch_tiles(const SharedTileArgs& a, bool fp8, hipStream_t stream) {
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)a.total), dim3(256), 0, stream, a); };
  fp8 ? launch(attn_fwd_kernel<D, E, 4, prefix_tile_keys(D), false, true, FP8>)
      : launch(attn_fwd_kernel<D, E, 4, prefix_tile_keys(D), false, true>);
  return hipGetLastError();
}

template <int D, class E, int WAYS>
hipError_t launch_merge_ways(MergeArgs a, int batch, hipStream_t stream) {
  constexpr int ROWS = 256 / (D / 4 * WAYS);
  a.chunks = (a.hq * a.nq + ROWS - 1) / ROWS;
  a.by_chunks = FastDiv::by(a.chunks);
  hipLaunchKernelGGL((shared_merge_kernel<D, E, WAYS>), dim3((unsigned)a.chunks * (unsigned)batch), dim3(256), 0, stream, a);
  return hipGetLastError();
}

template <int D, class E>
hipError_t launch_merge(const MergeArgs& a, int batch, int parts, hipStream_t stream) {
  // more than one round of CH partials: four threads share them, 4 each
  if (parts <= 8) return launch_merge_ways<D, E, 1>(a, batch, stream);
  return launch_merge_ways<D, E, 4>(a, batch, stream);
}

}  // namespace

SharedPlan plan_shared(const fa_fwd_params& p, const fa_shared_prefix& s, int page_size) {
  const int group = p.heads_q / p.heads_kv, rows = group * p.seqlen_q;
  SharedPlan plan{};
  plan.max_prefix = s.max_prefix_len / kPrefixUnit * kPrefixUnit;
  // (a prefix is cut at whole units: up to 63 of its keys go with each request's own)
  plan.max_suffix = s.max_suffix_len + kPrefixUnit - 1;
  const int64_t all_rows = (int64_t)p.batch * rows;
  const bool fp8 = p.kv_dtype == FA_DTYPE_FP8_E4M3;
  // (one group: exactly; several: each may leave a block unfilled, and the workgroups past the last block return)
  constexpr int block = 128;  // rows of a workgroup
  const int64_t group_blocks = s.num_groups > 1 ? all_rows / block + s.num_groups : (all_rows + block - 1) / block;
  plan.prefix_blocks = group_blocks;
  // Partitions.  A workgroup of the shared keys costs about 8 us before and after its tiles (64 keys in about 1 us at
  // D = 128, alone on its CU or one of two) and leaves 128 rows of partials; one a CU leaves the CU's other place to the
  // requests' own keys.  So: as many as there are CUs, half as many where those would have fewer than 1024 keys each (64
  // requests of 4 rows, 8 kv-heads, 8192 keys: the call takes 42 us at 512 keys, 37 at 1024; 32 of 16 rows, 16384 keys, 66
  // at 2048 and 86 at 4096; measured at D = 128 with one group only.  At D = 256 and with groups of 16, 24, 8 and 1 request it leaves
  // CUs empty: 162 working workgroups on 256).  A group has a block at least; which ones have more, and how long their
  // prefixes are, is not known here.  Own keys: 1024 waves, four a CU (512 at D = 256: 49 requests of up to 700 keys, 4 kv-heads, 55 us at 192
  // keys, 47 at 320), but no more than 576 keys each, for the last to start not to run on alone, and 320 where there are
  // many (256 requests of up to 1000 keys, 8 kv-heads, D = 64: 95 us whole, 91 at 576, 88 at 320; 32 of up to 2000: 66 at
  // 576, 72 at 320).
  constexpr int64_t kWgs = kCus, kLong = 1024, kWaves = 1024;
  auto whole = [](int64_t keys, int64_t parts) { return ((keys + parts - 1) / parts + kPrefixUnit - 1) / kPrefixUnit * kPrefixUnit; };
  // a partition spans a limited number of pages, and of FP8 scale blocks (not evened out afterwards: 4032 keys in pages of 16
  // are cut into 1984, 1984 and 64)
  auto fits = [&](int64_t len, int64_t pages) {
    len = std::min(len, (pages - 2) * page_size / kPrefixUnit * kPrefixUnit);
    return (int32_t)std::max<int64_t>(kPrefixUnit, fp8 ? std::min<int64_t>(len, kFp8Keys) : len);
  };
  const int64_t prefix_items = p.heads_kv * std::max<int64_t>((all_rows + block - 1) / block, s.num_groups);
  int64_t len = whole(plan.max_prefix, std::max<int64_t>(1, kWgs / prefix_items));
  if (len < kLong) len = std::min(kLong, whole(plan.max_prefix, std::max<int64_t>(1, kWgs / 2 / prefix_items)));
  plan.prefix_split = s.split_len > 0 ? s.split_len : fits(len, kPrefixPages);
  const int64_t suffix_items = (int64_t)p.batch * p.heads_kv * ((rows + 31) / 32);
  len = whole(plan.max_suffix, std::max<int64_t>(1, (p.head_dim == 256 ? kWaves / 2 : kWaves) / suffix_items));
  len = std::min<int64_t>(len, suffix_items <= kWaves / 4 ? 576 : 320);
  plan.suffix_split = s.split_len > 0 ? s.split_len : fits(len, kSuffixPages);
  plan.prefix_parts = (plan.max_prefix + plan.prefix_split - 1) / plan.prefix_split;
  plan.suffix_parts = (plan.max_suffix + plan.suffix_split - 1) / plan.suffix_split;
  return plan;
}

const char* shared_refusal(const fa_fwd_params& p, const fa_paged_kv& kv, const fa_shared_prefix& s) {
  const SharedPlan plan = plan_shared(p, s, kv.page_size);
  const int64_t rows = (int64_t)p.heads_q / p.heads_kv * p.seqlen_q;
  auto slots = [&](int64_t len) { return (len - 1) / kv.page_size + 2; };
  if (slots(plan.prefix_split) > kPrefixPages || slots(plan.suffix_split) > kSuffixPages)
    return "split_len too long for the page size: a partition may span at most 128 pages";
  if (p.kv_dtype == FA_DTYPE_FP8_E4M3 && s.split_len > kFp8Keys) return "split_len must be at most 4096 keys of FP8 pools";
  const int64_t out_rows = (int64_t)p.batch * p.heads_q * p.seqlen_q;
  if (out_rows > INT32_MAX / 2 || plan.prefix_blocks * p.heads_kv * plan.prefix_parts > INT32_MAX / 2 ||
      (int64_t)p.batch * p.heads_kv * plan.suffix_parts * ((rows + 31) / 32) > INT32_MAX / 2)
    return "grid too large";
  return nullptr;
}

size_t shared_workspace_bytes(const fa_fwd_params& p, const fa_paged_kv& kv, const fa_shared_prefix& s) {
  const SharedPlan plan = plan_shared(p, s, kv.page_size);
  return (size_t)p.batch * p.heads_q * p.seqlen_q * (size_t)(plan.prefix_parts + plan.suffix_parts) *
         ((size_t)p.head_dim + 2) * sizeof(float);
}

fa_status run_shared(const fa_fwd_params& p, const fa_paged_kv& kv, const fa_shared_prefix& s, void* workspace,
                     hipStream_t stream, const char** err) {
  const SharedPlan plan = plan_shared(p, s, kv.page_size);
  const bool fp8 = p.kv_dtype == FA_DTYPE_FP8_E4M3, bf = p.dtype == FA_DTYPE_BF16;
  const int64_t out_rows = (int64_t)p.batch * p.heads_q * p.seqlen_q;
  const int stride = plan.prefix_parts + plan.suffix_parts;
  SharedTileArgs a{};
  static_cast<TileArgs&>(a) = common_args(p);
  paged_args(a, kv);
  a.o = workspace;
  a.ml = (float*)workspace + out_rows * stride * p.head_dim;
  a.batch = p.batch;
  a.ppw = 1;
  a.shared.prefix_lens = s.prefix_lens;
  a.shared.cu_groups = s.cu_groups;
  a.shared.groups = s.cu_groups != nullptr ? s.num_groups : 1;
  a.shared.batch = p.batch;
  a.shared.max_prefix = s.max_prefix_len;
  a.shared.max_suffix = s.max_suffix_len;
  a.shared.table_keys = (int32_t)std::min<int64_t>((int64_t)kv.block_table_cols * kv.page_size, INT32_MAX);
  a.shared.part_stride = stride;
  a.shared.part_base = plan.prefix_parts;
  a.shared.prefix_split = plan.prefix_split;
  a.shared.suffix_split = plan.suffix_split;
  const int rows = a.group * p.seqlen_q;
  const int64_t prefix_wgs = plan.prefix_blocks * p.heads_kv * plan.prefix_parts;
  hipError_t e = hipSuccess;
  a.n_rowblk = (int32_t)plan.prefix_blocks;
  a.shared.suffix_blocks = (rows + 31) / 32;
  a.shared.by_page = FastDiv::by(kv.page_size);
  a.shared.by_hkv = FastDiv::by(p.heads_kv);
  a.shared.by_group = FastDiv::by(a.group);
  a.shared.by_nq = FastDiv::by(p.seqlen_q);
  a.shared.by_batch = FastDiv::by(p.batch);
  a.shared.by_prefix_blocks = FastDiv::by(a.n_rowblk);
  a.shared.by_suffix_blocks = FastDiv::by(a.shared.suffix_blocks);
  a.n_items = (int32_t)((int64_t)p.batch * p.heads_kv * plan.suffix_parts * a.shared.suffix_blocks);
  // The shared keys' workgroups go first; where the requests' own keys take longer (an estimate: 0.65 us a tile and CU of the
  // former, D = 128's, 4.5 TB/s for half of the longest of the latter), only one a CU, the rest behind the own keys' (256 requests of
  // up to 1000 keys behind 4080, D = 64: 82 us, 79 so; FP8, 128 of up to 700 behind 32768: 174, 183 so).
  const double prefix_us = 0.65 * plan.prefix_blocks * p.heads_kv * (plan.max_prefix / 64.0) / kCus;
  const double suffix_us = (double)p.batch * p.heads_kv * plan.max_suffix * p.head_dim * (fp8 ? 1 : 2) / 4.5e6;
  a.shared.prefix_first = (int32_t)(suffix_us > prefix_us ? std::min<int64_t>(prefix_wgs, kCus) : prefix_wgs);
  a.shared.suffix_wgs = (int32_t)(((int64_t)a.n_items + 3) / 4);
  a.total = (int32_t)(prefix_wgs + a.shared.suffix_wgs);
  e = by_dim_and_type(p.head_dim, bf, [&](auto d, auto t) { return launch_tiles<decltype(d)::value, decltype(t)>(a, fp8, stream); });
  if (e != hipSuccess) return hip_status(e, err);

  MergeArgs m{};
  m.part = (float*)a.o;
  m.ml = a.ml;
  m.o = p.o;
  m.lse = p.lse;
  m.sob = p.o_stride_b;
  m.soh = p.o_stride_h;
  m.son = p.o_stride_n;
  m.slb = p.lse_stride_b;
  m.slh = p.lse_stride_h;
  m.seqlens = kv.seqlens_k;
  m.hq = p.heads_q;
  m.nq = p.seqlen_q;
  m.by_prefix_split = FastDiv::by(plan.prefix_split);
  m.by_suffix_split = FastDiv::by(plan.suffix_split);
  m.causal = p.causal;
  m.shared = a.shared;
  m.tile = a;
  m.fp8 = fp8;
  e = by_dim_and_type(p.head_dim, bf, [&](auto d, auto t) {
    return launch_merge<decltype(d)::value, decltype(t)>(m, p.batch, stride, stream);
  });
  return hip_status(e, err);
}

}  // namespace fa
