// 4-bit K/V cache rows: the writer (bulk, and single tokens into a cache), and the reader back to floats.
//
// A row is one token of one kv-head, x[D].  It is held as D codes of 4 bits between its ends:
//   zero  = fp16(lo), scale = fp16((hi - lo) * fp32(1/15))     lo, hi = min, max of the row, held to +-65504
//   code  = clamp(rint((x - zero) / scale), 0, 15)             in fp32, halves to even; 0 where scale is 0
//   value = code * scale + zero
// The codes are taken against the rounded scale and zero, so rounding those costs nothing but the clamp at the
// ends.  fp16 for the pair: 4 bytes a row (6% of it at D=128), 2^-11 of the row's ends against the 2^-5 of the
// range that a code is off by.  A NaN in a row makes its scale and zero NaN; infinities become the row's ends.
//
// Two codes a byte, the even channel in the low half, channels in order: a row is D/2 contiguous bytes, and the
// (scale, zero) pairs lie in a tensor of their own, one 4-byte word a row.  Scales per row (not per block of
// keys) let rows be appended and picked one at a time.
//
// A lane holds 8 channels (16 bytes of 16-bit input, one 4-byte word of codes), so D/8 lanes hold a row and its ends are a
// reduction over them; UNROLL rows a lane are loaded before any is worked on.  16 x 8 x 32768 rows of D=128 bf16 (1.36 GB
// each way): written in 251 us, read back in 223, 5.4 and 6.1 TB/s (265 and 234 under the profiler).  The reader is bound by
// HBM; the writer by the vector unit as well, which its 154 instructions for 8 channels a lane keep busy nearly all the time.
#include "fa_device.hpp"
#include "fa_internal.hpp"

namespace fa {

namespace {

constexpr float kF16Max = 65504.f;
constexpr int kBlock = 256;

template <class T>
struct Chunk {  // 8 channels as read from memory
  u32x4 w[sizeof(T) / 2];
};

template <class T>
__device__ __forceinline__ Chunk<T> load_chunk(const T* p) {
  Chunk<T> c;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) c.w[i] = __builtin_nontemporal_load((const u32x4*)p + i);
  return c;
}

template <class T>
__device__ __forceinline__ float chunk_value(const Chunk<T>& c, int e) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(c.w[e / 4][e % 4]);
  } else {
    using Tag = typename std::conditional<std::is_same<T, __bf16>::value, BF16, F16>::type;
    const uint32_t w = c.w[0][e / 2];
    return (e & 1) ? hi_f32<Tag>(w) : lo_f32<Tag>(w);
  }
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float vmin(float a, float b) { return __builtin_elementwise_minimum(a, b); }

// x as an fp32 value of its own: without it a product that is then rounded to fp16 becomes one mixed-precision
// instruction with a single rounding, and the definition (and the torch form) rounds twice.
__device__ __forceinline__ float rounded(float x) {
  __asm__("" : "+v"(x));
  return x;
}

// Minimum and maximum over the LPR (8, 16 or 32) lanes that hold a row; NaN wins.  Exchanges inside 16 lanes are
// DPP moves (neighbour, pair, then the mirrored half and row, whose lanes already agree), the 16-lane one a shuffle.
template <int LPR>
__device__ __forceinline__ void row_ends(float& lo, float& hi) {
  lo = vmin(lo, dpp<0xB1>(lo)), hi = vmax(hi, dpp<0xB1>(hi));    // quad_perm [1,0,3,2]
  lo = vmin(lo, dpp<0x4E>(lo)), hi = vmax(hi, dpp<0x4E>(hi));    // quad_perm [2,3,0,1]
  lo = vmin(lo, dpp<0x141>(lo)), hi = vmax(hi, dpp<0x141>(hi));  // row_half_mirror
  if constexpr (LPR >= 16) lo = vmin(lo, dpp<0x140>(lo)), hi = vmax(hi, dpp<0x140>(hi));  // row_mirror
  if constexpr (LPR >= 32) lo = vmin(lo, __shfl_xor(lo, 16)), hi = vmax(hi, __shfl_xor(hi, 16));
}

// x / scale for 0 <= x <= 16 scale and a positive scale, correctly rounded wherever the quotient is normal: the product
// with y = RN(1 / scale) and one residual step (Markstein).  A quotient too small to be normal rounds to code 0 either
// way.  (A larger x could overflow the product, and the residual step make a NaN of it.)
__device__ __forceinline__ float div_scale(float x, float scale, float y) {
  const float q = x * y;
  return __builtin_fmaf(__builtin_fmaf(-q, scale, x), y, q);
}

// Codes of the 8 channels of a lane, and the row's (scale, zero) word.  Every lane of a row is active.
template <class T, int LPR>
__device__ __forceinline__ uint32_t encode(const Chunk<T>& c, uint32_t& pair) {
  float x[8], lo, hi;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = chunk_value<T>(c, e);
  lo = hi = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) lo = vmin(lo, x[e]), hi = vmax(hi, x[e]);
  row_ends<LPR>(lo, hi);
  lo = vmin(vmax(lo, -kF16Max), kF16Max);
  hi = vmin(vmax(hi, -kF16Max), kF16Max);
  const f16x2 sz = {(_Float16)rounded((hi - lo) * (1.0f / 15.0f)), (_Float16)lo};
  pair = __builtin_bit_cast(uint32_t, sz);
  const float scale = (float)sz[0], zero = (float)sz[1];
  uint32_t codes = 0;
  if (scale > 0.f) {
    const float y = __fdiv_rn(1.0f, scale);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // held to where the code already is 0 or 15, infinities among them (16 scale is exact)
      const float d = __builtin_amdgcn_fmed3f(x[e] - zero, 0.f, 16.f * scale);
      codes |= (uint32_t)fminf(__builtin_rintf(div_scale(d, scale, y)), 15.f) << (4 * e);
    }
  }
  return codes;
}

// Where the rows of a lane are.  A workgroup takes UNROLL * RPS rows, RPS a step: those of one (batch, head) from n0 on,
// or where a head has fewer rows than half of that (FLAT: pages, single tokens) those of the flattened [B, H, N], at two
// divisions a row (2053 pages of 8 heads x 16 tokens, D=64: read in 9 us, 12 without; 16 x 8 x 32768 rows: written in
// 311 us, 250 without).
template <bool FLAT, int RPS, int UNROLL>
struct RowPlace {
  int b[UNROLL], h[UNROLL], n[UNROLL];
  bool ok[UNROLL];
  __device__ __forceinline__ RowPlace(const Int4Args& a, int first) {
    if constexpr (FLAT) {
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int64_t row = (int64_t)blockIdx.x * (RPS * UNROLL) + first + u * RPS;
        ok[u] = row < a.rows;
        const uint32_t r = ok[u] ? (uint32_t)row : 0u, bh = r / (uint32_t)a.n;
        n[u] = (int)(r - bh * (uint32_t)a.n);
        b[u] = (int)(bh / (uint32_t)a.h);
        h[u] = (int)(bh - (uint32_t)b[u] * (uint32_t)a.h);
      }
    } else {
      const uint32_t bh = blockIdx.x / (uint32_t)a.chunks, b0 = bh / (uint32_t)a.h;
      const int n0 = (int)(blockIdx.x - bh * (uint32_t)a.chunks) * (RPS * UNROLL) + first;
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        b[u] = (int)b0;
        h[u] = (int)(bh - b0 * (uint32_t)a.h);
        n[u] = n0 + u * RPS;
        ok[u] = n[u] < a.n;
      }
    }
  }
  __device__ __forceinline__ int64_t at(int u, int64_t sb, int64_t sh, int64_t sn) const {
    return b[u] * sb + h[u] * sh + n[u] * sn;
  }
};

// Bulk writer.
template <class T, int D, int UNROLL, bool FLAT>
__global__ void __launch_bounds__(kBlock) quantize_kv_int4_kernel(const Int4Args a) {
  constexpr int LPR = D / 8, RPS = kBlock / LPR;  // lanes a row, rows a step
  const int lane = (int)threadIdx.x % LPR;
  const RowPlace<FLAT, RPS, UNROLL> at(a, (int)threadIdx.x / LPR);
  Chunk<T> c[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    if (at.ok[u]) c[u] = load_chunk((const T*)a.x + at.at(u, a.sxb, a.sxh, a.sxn) + 8 * lane);
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    if (!at.ok[u]) return;  // whole rows: their lanes leave together
    uint32_t pair;
    const uint32_t w = encode<T, LPR>(c[u], pair);
    *(uint32_t*)(a.codes + at.at(u, a.scb, a.sch, a.scn) + 4 * lane) = w;
    if (lane == 0) a.pairs[at.at(u, a.ssb, a.ssh, a.ssn)] = pair;
  }
}

// The reader: floats from codes.  code * scale is exact in fp32, so a value takes one rounding there and one to T.
template <class T, int D, int UNROLL, bool FLAT>
__global__ void __launch_bounds__(kBlock) dequantize_kv_int4_kernel(const Int4Args a) {
  constexpr int LPR = D / 8, RPS = kBlock / LPR;
  const int lane = (int)threadIdx.x % LPR;
  const RowPlace<FLAT, RPS, UNROLL> at(a, (int)threadIdx.x / LPR);
  uint32_t w[UNROLL], pair[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    if (at.ok[u]) {
      w[u] = *(const uint32_t*)(a.codes + at.at(u, a.scb, a.sch, a.scn) + 4 * lane);
      pair[u] = a.pairs[at.at(u, a.ssb, a.ssh, a.ssn)];
    }
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    if (!at.ok[u]) return;
    const float scale = lo_f32<F16>(pair[u]), zero = hi_f32<F16>(pair[u]);
    T* out = (T*)a.x + at.at(u, a.sxb, a.sxh, a.sxn) + 8 * lane;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = rounded(__builtin_fmaf((float)((w[u] >> (4 * e)) & 15u), scale, zero));
    if constexpr (sizeof(T) == 4) {
      __builtin_nontemporal_store(u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                                        __float_as_uint(v[3])}, (u32x4*)out);
      __builtin_nontemporal_store(u32x4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]),
                                        __float_as_uint(v[7])}, (u32x4*)out + 1);
    } else {
      using Tag = typename std::conditional<std::is_same<T, __bf16>::value, BF16, F16>::type;
      __builtin_nontemporal_store(u32x4{pack2<Tag>(v[0], v[1]), pack2<Tag>(v[2], v[3]), pack2<Tag>(v[4], v[5]),
                                        pack2<Tag>(v[6], v[7])}, (u32x4*)out);
    }
  }
}

// New tokens into a cache: token i of sequence b goes to position seqlens_k[b] + i, K and V in one launch (they are
// few rows, and the launch is most of the time).  Tokens whose position lies outside the cache, or whose page lies
// outside the pool, are not written.
template <class T, int D>
__global__ void __launch_bounds__(kBlock) append_kv_int4_kernel(const AppendArgs a) {
  constexpr int LPR = D / 8, RPS = kBlock / LPR;
  const int lane = (int)threadIdx.x % LPR;
  const Int4Args& t = blockIdx.y == 0 ? a.k : a.v;
  const int64_t row = (int64_t)blockIdx.x * RPS + (int)threadIdx.x / LPR;
  if (row >= t.rows) return;
  const uint32_t bh = (uint32_t)row / (uint32_t)t.n;
  const int n = (int)((uint32_t)row - bh * (uint32_t)t.n), b = (int)(bh / (uint32_t)t.h);
  const int h = (int)(bh - (uint32_t)b * (uint32_t)t.h);
  const Chunk<T> c = load_chunk((const T*)t.x + b * t.sxb + h * t.sxh + n * t.sxn + 8 * lane);
  uint32_t pair;
  const uint32_t codes = encode<T, LPR>(c, pair);
  const int64_t pos = (int64_t)a.seqlens_k[b] + n;
  if (pos < 0 || pos >= a.capacity) return;
  int64_t at = b, slot = pos;
  if (a.block_table != nullptr) {
    at = a.block_table[b * a.sbt + pos / a.page_size];
    slot = pos % a.page_size;
    if (at < 0 || at >= a.num_pages) return;
  }
  *(uint32_t*)(t.codes + at * t.scb + h * t.sch + slot * t.scn + 4 * lane) = codes;
  if (lane == 0) t.pairs[at * t.ssb + h * t.ssh + slot * t.ssn] = pair;
}

Int4Args int4_args(const fa_int4_params& p) {
  Int4Args a{};
  a.x = p.x;
  a.sxb = p.x_stride_b;
  a.sxh = p.x_stride_h;
  a.sxn = p.x_stride_n;
  a.codes = (uint8_t*)p.codes;
  a.scb = p.codes_stride_b;
  a.sch = p.codes_stride_h;
  a.scn = p.codes_stride_n;
  a.pairs = (uint32_t*)p.scale;
  a.ssb = p.scale_stride_b;
  a.ssh = p.scale_stride_h;
  a.ssn = p.scale_stride_n;
  a.h = p.heads;
  a.n = p.seqlen;
  a.rows = (int64_t)p.batch * p.heads * p.seqlen;
  return a;
}

constexpr int kUnroll = 4;

template <class T, int D>
hipError_t launch_rows(Int4Args a, bool read, hipStream_t stream, const char** err) {
  constexpr int per = kBlock / (D / 8) * kUnroll;
  const bool flat = a.n < per / 2 && a.rows <= INT32_MAX;
  a.chunks = (a.n - 1) / per + 1;
  const int64_t blocks = flat ? (a.rows + per - 1) / per : a.rows / a.n * a.chunks;
  if (blocks > INT32_MAX) {
    *err = "too many rows";
    return hipErrorInvalidConfiguration;
  }
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kBlock), 0, stream, a); };
  if (read) {
    flat ? launch(dequantize_kv_int4_kernel<T, D, kUnroll, true>) : launch(dequantize_kv_int4_kernel<T, D, kUnroll, false>);
  } else {
    flat ? launch(quantize_kv_int4_kernel<T, D, kUnroll, true>) : launch(quantize_kv_int4_kernel<T, D, kUnroll, false>);
  }
  return hipGetLastError();
}

template <class T, int D>
hipError_t launch_append(const AppendArgs& a, hipStream_t stream) {
  constexpr int per = kBlock / (D / 8);
  hipLaunchKernelGGL((append_kv_int4_kernel<T, D>), dim3((unsigned)((a.k.rows + per - 1) / per), 2), dim3(kBlock), 0,
                     stream, a);
  return hipGetLastError();
}

template <class F>
hipError_t by_type(int dtype, int d, F&& f) {
  auto dim = [&](auto t) {
    using T = decltype(t);
    return d == 64 ? f(t, std::integral_constant<int, 64>{})
                   : d == 128 ? f(T{}, std::integral_constant<int, 128>{}) : f(T{}, std::integral_constant<int, 256>{});
  };
  return dtype == FA_DTYPE_BF16 ? dim(__bf16{}) : dtype == FA_DTYPE_F16 ? dim(_Float16{}) : dim(float{});
}

}  // namespace

fa_status run_int4_rows(const fa_int4_params& p, bool read, hipStream_t stream, const char** err) {
  const Int4Args a = int4_args(p);
  if (p.seqlen > (1 << 30)) {
    *err = "too many rows";
    return FA_ERR_UNSUPPORTED;
  }
  return hip_status(by_type(p.dtype, p.head_dim, [&](auto t, auto d) {
    return launch_rows<decltype(t), decltype(d)::value>(a, read, stream, err);
  }), err);
}

fa_status run_append_int4(const fa_int4_append_params& p, hipStream_t stream, const char** err) {
  AppendArgs a{};
  a.k = int4_args(p.k);
  a.v = int4_args(p.v);
  a.seqlens_k = p.seqlens_k;
  a.block_table = p.block_table;
  a.sbt = p.block_table_stride;
  a.page_size = p.page_size;
  a.num_pages = p.num_pages;
  a.capacity = p.block_table != nullptr ? (int64_t)p.block_table_cols * p.page_size : p.capacity;
  if (a.k.rows > INT32_MAX - kBlock) {
    *err = "too many rows";
    return FA_ERR_UNSUPPORTED;
  }
  return hip_status(by_type(p.k.dtype, p.k.head_dim, [&](auto t, auto d) {
    return launch_append<decltype(t), decltype(d)::value>(a, stream);
  }), err);
}

}  // namespace fa
