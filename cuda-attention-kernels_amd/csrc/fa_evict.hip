// Eviction from a K/V cache by accumulated attention weight: which keys stay, and their rows moved together.
//
// Per (sequence, kv-head), with n keys in the cache and room for `keep`: all keys where n <= keep; else the last
// `recent` ones and, of the others, the keep - recent with the highest scores (equal scores: the lower index; a NaN
// counts as the highest, -0 as 0), in their order in the cache.
//
//   * evict_select_kernel: one workgroup a (sequence, kv-head).  The threshold is found digit by digit: scores map to
//     unsigned integers of the same order, and four passes each count the 8-bit digits of the candidates that share
//     the digits found so far.  The counters are 32 copies, lane l using copy l % 32, which is also its LDS bank:
//     scores of a softmax crowd into few exponents, and 64 lanes adding to one counter would take 64 turns.  Integer
//     counts: the result does not depend on the order of the additions.  A last pass writes the indices in order (the
//     candidates above the threshold and the first of those equal to it).  The scores are read five times, from the
//     L2 after the first: 4 bytes a key against the rows of 8 to 1000 that the gather moves.
//   * gather_rows_kernel: rows of up to kMaxEvictTensors tensors in one launch; a thread copies units of the widest
//     power of two (16 bytes at most) that a tensor's rows, strides and addresses allow.  HBM-bound.
#include "fa_device.hpp"
#include "fa_internal.hpp"

namespace fa {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kItems = 4;
constexpr int kCopies = 32;

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // rows of scores start at any float

// Unsigned integers in the order of the scores: NaN above +inf, -0 equal to 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  if (x != x) return 0xffffffffu;
  if (u == 0x80000000u) return 0x80000000u;
  return (u >> 31) ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kThreads) evict_select_kernel(const EvictArgs a) {
  __shared__ uint32_t hist[256 * kCopies];
  __shared__ uint32_t total[256];
  __shared__ uint32_t found[2];  // this pass's digit, and how many are still wanted among its candidates
  __shared__ uint32_t wave_sum[2][kWaves];

  const int bh = (int)blockIdx.x, b = bh / a.h, h = bh - b * a.h;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = a.seqlens_k != nullptr ? min(max(a.seqlens_k[b], 0), a.nk) : a.nk;
  const float* s = a.scores + b * a.ssb + h * a.ssh;
  int32_t* index = a.index + (int64_t)bh * a.keep;
  float* out = a.scores_out + (int64_t)bh * a.keep;
  if (h == 0 && tid == 0) a.seqlens_out[b] = min(n, a.keep);

  if (n <= a.keep) {
    for (int j = tid; j < a.keep; j += kThreads) {
      index[j] = j < n ? j : -1;
      out[j] = j < n ? s[j] : 0.f;
    }
    return;
  }
  const int old = n - a.recent, want = a.keep - a.recent;  // 0 <= recent <= keep < n
  for (int j = tid; j < a.recent; j += kThreads) {
    index[want + j] = old + j;
    out[want + j] = s[old + j];
  }
  if (want == 0) return;

  // ---- the key of rank `want` among the candidates [0, old) ------------------------------------------------
  uint32_t prefix = 0, rank = (uint32_t)want;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256 * kCopies; i += kThreads) hist[i] = 0;
    __syncthreads();
    const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    auto count = [&](float x) __attribute__((always_inline)) {
      const uint32_t k = order_key(x);
      if ((k & mask) == prefix) atomicAdd(&hist[((k >> shift) & 255u) * kCopies + (lane & (kCopies - 1))], 1u);
    };
    const int whole = old & ~(kItems - 1);
    for (int j = tid * kItems; j < whole; j += kThreads * kItems) {
      const f32x4u x = *(const f32x4u*)(s + j);
#pragma unroll
      for (int e = 0; e < kItems; ++e) count(x[e]);
    }
    if (whole + tid < old) count(s[whole + tid]);
    __syncthreads();
    if (tid < 256) {
      uint32_t t = 0;
#pragma unroll 8
      for (int i = 0; i < kCopies; ++i) t += hist[tid * kCopies + ((i + tid) & (kCopies - 1))];  // a bank each
      total[tid] = t;
    }
    __syncthreads();
    if (wave == 0) {
      // lane l holds digits 255 - 4l .. 252 - 4l: running counts from the highest digit down
      uint32_t c[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += c[i] = total[255 - 4 * lane - i];
      uint32_t upto = sum;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const uint32_t t = __shfl_up(upto, off);
        if (lane >= off) upto += t;
      }
      uint32_t above = upto - sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (above < rank && above + c[i] >= rank) {  // one lane and digit: the candidates hold at least `rank`
          found[0] = (uint32_t)(255 - 4 * lane - i);
          found[1] = rank - above;
        }
        above += c[i];
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    rank = found[1];
  }

  // ---- indices in order: keys above `prefix`, and the first `rank` equal to it ------------------------------
  uint32_t above = 0, equal = 0;  // of the chunks done
  int buf = 0;
  for (int j0 = 0; j0 < old; j0 += kThreads * kItems, buf ^= 1) {
    const int j = j0 + tid * kItems;
    float x[kItems];
    if (j + kItems <= old) {
      const f32x4u v = *(const f32x4u*)(s + j);
#pragma unroll
      for (int e = 0; e < kItems; ++e) x[e] = v[e];
    } else {
#pragma unroll
      for (int e = 0; e < kItems; ++e) x[e] = j + e < old ? s[j + e] : 0.f;
    }
    uint32_t flag[kItems], sum = 0;  // above in the low half, equal in the high half (a chunk holds 4096)
#pragma unroll
    for (int e = 0; e < kItems; ++e) {
      const uint32_t k = order_key(x[e]);
      flag[e] = j + e >= old ? 0u : k > prefix ? 1u : k == prefix ? 0x10000u : 0u;
      sum += flag[e];
    }
    uint32_t upto = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t t = __shfl_up(upto, off);
      if (lane >= off) upto += t;
    }
    if (lane == 63) wave_sum[buf][wave] = upto;
    __syncthreads();  // (the buffers alternate: one barrier a chunk)
    uint32_t before = upto - sum, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t t = wave_sum[buf][w];
      if (w < wave) before += t;
      all += t;
    }
    uint32_t na = above + (before & 0xffffu), ne = equal + (before >> 16);
#pragma unroll
    for (int e = 0; e < kItems; ++e) {
      if (flag[e] == 1u || (flag[e] != 0u && ne < rank)) {
        const uint32_t pos = na + min(ne, rank);
        index[pos] = j + e;
        out[pos] = x[e];
      }
      na += flag[e] & 0xffffu;
      ne += flag[e] >> 16;
    }
    above += all & 0xffffu;
    equal += all >> 16;
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
  U v[STEP];
  char* to[STEP];
#pragma unroll
  for (int i = 0; i < STEP; ++i) {
    const uint32_t u = u0 + 256 * i;
    to[i] = nullptr;
    if (u < all) {
      const uint32_t r = t.shift >= 0 ? u >> t.shift : u / units, c = u - r * units;
      const int j = index[r];
      to[i] = dst + r * t.dn + c * sizeof(U);
      v[i] = U{};
      if (j >= 0) v[i] = *(const U*)(src + j * t.sn + c * sizeof(U));
    }
  }
#pragma unroll
  for (int i = 0; i < STEP; ++i) {
    if (to[i] != nullptr) *(U*)to[i] = v[i];
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
  a.scores_out = p.scores_out;
  a.seqlens_out = p.seqlens_out;
  a.h = p.heads;
  a.nk = p.seqlen;
  a.keep = p.keep;
  a.recent = p.recent;
  const int64_t bh = (int64_t)p.batch * p.heads;
  int64_t units = 0;  // most of any tensor, per (sequence, kv-head)
  for (int i = 0; i < p.num_tensors; ++i) {
    const fa_evict_tensor& t = p.tensors[i];
    EvictTensor& g = a.tensors[i];
    g = EvictTensor{t.src, t.dst, t.src_stride_b, t.src_stride_h, t.src_stride_n, t.dst_stride_b, t.dst_stride_h,
                    t.dst_stride_n, 0, 0, -1};
    const uint64_t bits = (uint64_t)(uintptr_t)t.src | (uint64_t)(uintptr_t)t.dst | (uint64_t)t.row_bytes |
                          (uint64_t)t.src_stride_b | (uint64_t)t.src_stride_h | (uint64_t)t.src_stride_n |
                          (uint64_t)t.dst_stride_b | (uint64_t)t.dst_stride_h | (uint64_t)t.dst_stride_n | 16u;
    g.unit = (int32_t)(bits & (~bits + 1));  // the lowest set bit
    g.units = (int32_t)(t.row_bytes / g.unit);
    for (int s = 0; s < 31; ++s) {
      if ((int64_t{1} << s) == g.units) g.shift = s;
    }
    units = units > (int64_t)p.keep * g.units ? units : (int64_t)p.keep * g.units;
  }
  a.chunks = (int32_t)((units + 1023) / 1024);
  if (units > INT32_MAX - 1024 || bh * a.chunks > INT32_MAX || bh > INT32_MAX) {
    *err = "grid too large";
    return FA_ERR_UNSUPPORTED;
  }
  hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)bh), dim3(kThreads), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.chunks == 0) return hip_status(e, err);
  hipLaunchKernelGGL(gather_rows_kernel, dim3((unsigned)(bh * a.chunks), (unsigned)p.num_tensors), dim3(256), 0, stream,
                     a);
  return hip_status(hipGetLastError(), err);
}

}  // namespace fa
