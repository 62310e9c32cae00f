// Native dispatcher kernels of the custom op fused_attn::attention for GPU tensors.
//
// The op is defined in Python (fused_attn/ops.py), whose kernel checks, prepares and launches a call through
// ctypes: 20-27 us of host time, more than the GPU needs for a small call.  The kernels here take the calls
// that need no preparation (operands the HIP kernels read as they are, no backend forced by the environment, a
// device the Python side has found supported) and launch them in 6-8 us; every other call, errors included,
// goes on to the Python kernels, which stay the one place that says what is accepted and how it fails.
//
// The choice of kernel and partitions repeats ops._hip_kernel_for and ops.default_split_len
// (fa_torch_route lets a test compare the two).
//
// fa_torch_functions gives functions that do the same for attention_shared_prefix, allocate_pages, release_pages and
// append_kv_paged, which are no ops: they take Python objects, and return None for what the Python code is to handle.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <initializer_list>
#include <vector>

#include "../../include/fused_attn_hip.h"

namespace {

// C ABI of the HIP library, set once by fa_torch_bind (ctypes has loaded the library, maybe from a path the
// user named), and the devices the Python side has found supported.
struct Abi {
  size_t (*fwd_workspace_bytes)(const fa_fwd_params*);
  fa_status (*fwd_ws)(const fa_fwd_params*, void*, size_t, void*);
  size_t (*splitk_workspace_bytes)(int32_t, int32_t, int32_t, int32_t, int32_t);
  fa_status (*splitk)(const fa_fwd_params*, int32_t, void*, size_t, void*);
  const char* (*last_error)();
};
Abi g_abi{};
struct SharedAbi {
  size_t (*workspace_bytes)(const fa_fwd_params*, const fa_paged_kv*, const fa_shared_prefix*);
  fa_status (*call)(const fa_fwd_params*, const fa_paged_kv*, const fa_shared_prefix*, void*, size_t, void*);
};
SharedAbi g_shared{};
struct PagesAbi {
  fa_status (*allocate)(const fa_pages_params*, void*);
  fa_status (*release)(const fa_pages_params*, void*);
  fa_status (*append)(const fa_append_paged_params*, void*);
};
PagesAbi g_pages{};
std::atomic<uint64_t> g_devices{0};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool is_short_decode(int64_t b, int64_t hq, int64_t hkv, int64_t nq, int64_t nk, int64_t d) {
  const int64_t group = hq / hkv, heads = b * hq;
  if (nq == 0 || group * nq > 32 || nq > 8) return false;
  if (heads <= 64) return d != 256 && (group > 1 || nq <= 4) && nk >= (d == 64 ? 641 : 512);
  const bool many = heads > (d == 256 ? 256 : 512);
  if (group < 4) {
    if (group == 1 || nq > 4) return false;
    if (nq > 2) return nk >= 1600;
    if (many) return nk >= (d == 64 ? 384 : 192);
    return nk >= (d == 64 ? 1000 : d == 128 ? 768 : 512);
  }
  if (nq > 4) return nk >= (d == 64 ? 1600 : 1280);
  if (many) return nk >= (d != 64 ? 192 : nq <= 2 ? 256 : 512);
  return nk >= (d != 64 ? 512 : nq <= 2 ? 641 : 1000);
}

// Keys per split-K partition, or 0 for the prefill kernel.
int64_t route(bool half, int64_t b, int64_t hq, int64_t hkv, int64_t nq, int64_t nk, int64_t d) {
  if (!half || !(d == 64 || d == 128 || d == 256)) return 0;
  if (!(nq <= 16 && nk >= 2048) && !is_short_decode(b, hq, hkv, nq, nk, d)) return 0;
  const int64_t items = std::max<int64_t>(1, b * hkv * ceil_div(hq / hkv * nq, 128));
  const int64_t parts = std::max<int64_t>(1, ceil_div(2048, items));
  const int64_t keys = ceil_div(ceil_div(std::max<int64_t>(nk, 1), parts), 64) * 64;
  return std::min<int64_t>(std::max<int64_t>(keys, 128), 4096);
}

// The kernels read t as it is: unit stride along D, 16-byte aligned rows, token strides below 16 MiB.
bool readable(const at::Tensor& t) {
  if (t.stride(3) != 1 || reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 != 0) return false;
  for (int i = 0; i < 3; ++i) {
    if (t.size(i) > 1 && t.stride(i) % 8 != 0) return false;
  }
  return t.size(2) <= 1 || t.stride(2) * (int64_t)t.element_size() < (int64_t{1} << 24);
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return FA_DTYPE_F16;
    case at::kBFloat16: return FA_DTYPE_BF16;
    case at::kFloat: return FA_DTYPE_F32;
    default: return -1;
  }
}

// Whether the environment names a backend.  Read with the GIL held (torch calls kernels without it): os.environ sets
// variables under it, and a setenv beside this getenv may move the table it reads.
bool backend_forced() {
  const PyGILState_STATE gil = PyGILState_Ensure();
  const char* forced = std::getenv("FUSED_ATTN_BACKEND");
  const bool set = forced != nullptr && *forced != '\0';
  PyGILState_Release(gil);
  return set;
}

bool takes(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || !q.is_cuda() || !k.is_cuda() || !v.is_cuda()) return false;
  const int dev = q.device().index();
  if (dev < 0 || dev >= 64 || !((g_devices.load(std::memory_order_acquire) >> dev) & 1)) return false;
  if (k.device() != q.device() || v.device() != q.device()) return false;
  if (q.layout() != at::kStrided || k.layout() != at::kStrided || v.layout() != at::kStrided) return false;
  if (dtype_code(q.scalar_type()) < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) return false;
  if (!k.sizes().equals(v.sizes()) || k.size(3) != q.size(3) || (k.size(0) != q.size(0) && k.size(0) != 1)) return false;
  if (q.numel() == 0 || k.numel() == 0 || q.size(1) % k.size(1) != 0) return false;
  for (const at::Tensor* t : {&q, &k}) {
    for (const int64_t n : t->sizes()) {
      if (n > INT32_MAX) return false;
    }
  }
  if (!readable(q) || !readable(k) || !readable(v)) return false;
  return !backend_forced();
}

const c10::OperatorHandle& attention_op() {
  static const c10::OperatorHandle op = c10::Dispatcher::singleton().findSchemaOrThrow("fused_attn::attention", "");
  return op;
}

// The Python kernel registered under `key`.
at::Tensor call_python(c10::DispatchKey key, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool causal,
                       std::optional<double> scale) {
  torch::jit::Stack stack;
  torch::jit::push(stack, q, k, v, causal, scale);
  attention_op().callBoxedForDispatchKey(key, stack);
  return torch::jit::pop(stack).toTensor();
}

at::Tensor attention_gpu(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool causal,
                         std::optional<double> scale) {
  if (!takes(q, k, v)) return call_python(c10::DispatchKey::CompositeExplicitAutograd, q, k, v, causal, scale);
  const c10::DeviceGuard guard(q.device());
  at::Tensor o = at::empty(q.sizes(), q.options());
  fa_fwd_params p{};
  auto strides = [](const at::Tensor& t, int64_t& b, int64_t& h, int64_t& n) {
    b = t.size(0) > 1 ? t.stride(0) : 0;  // a dimension of size 1 is never stepped over
    h = t.size(1) > 1 ? t.stride(1) : 0;
    n = t.size(2) > 1 ? t.stride(2) : 0;
  };
  p.q = q.const_data_ptr();
  p.k = k.const_data_ptr();
  p.v = v.const_data_ptr();
  p.o = o.mutable_data_ptr();
  strides(q, p.q_stride_b, p.q_stride_h, p.q_stride_n);
  strides(k, p.k_stride_b, p.k_stride_h, p.k_stride_n);
  strides(v, p.v_stride_b, p.v_stride_h, p.v_stride_n);
  strides(o, p.o_stride_b, p.o_stride_h, p.o_stride_n);
  p.batch = (int32_t)q.size(0);
  p.heads_q = (int32_t)q.size(1);
  p.heads_kv = (int32_t)k.size(1);
  p.seqlen_q = (int32_t)q.size(2);
  p.seqlen_k = (int32_t)k.size(2);
  p.head_dim = (int32_t)q.size(3);
  p.scale = (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)q.size(3)));
  p.causal = causal ? 1 : 0;
  p.dtype = p.kv_dtype = (decltype(p.dtype))dtype_code(q.scalar_type());
  void* stream = at::hip::getCurrentHIPStreamMasqueradingAsCUDA(q.device().index()).stream();
  auto workspace = [&](size_t bytes) { return at::empty({(int64_t)(bytes / 4)}, q.options().dtype(at::kFloat)); };

  const int64_t split_len = route(q.scalar_type() != at::kFloat, p.batch, p.heads_q, p.heads_kv, p.seqlen_q, p.seqlen_k, p.head_dim);
  fa_status st;
  if (split_len > 0) {
    const size_t need = g_abi.splitk_workspace_bytes(p.batch, p.heads_q, p.seqlen_q, p.head_dim,
                                                     (int32_t)ceil_div(p.seqlen_k, split_len));
    const at::Tensor ws = workspace(need);
    st = g_abi.splitk(&p, (int32_t)split_len, ws.mutable_data_ptr(), need, stream);
  } else {
    const size_t need = g_abi.fwd_workspace_bytes(&p);
    const at::Tensor ws = need ? workspace(need) : at::Tensor();
    st = g_abi.fwd_ws(&p, need ? ws.mutable_data_ptr() : nullptr, need, stream);
  }
  TORCH_CHECK(st != FA_ERR_HIP, "fused_attn HIP ", split_len > 0 ? "attention_splitk" : "attention_fwd", " failed (HIP error): ",
              g_abi.last_error());
  // refused before anything was launched: the Python kernel reports it
  if (st != FA_OK) return call_python(c10::DispatchKey::CompositeExplicitAutograd, q, k, v, causal, scale);
  return o;
}

// Rows of whole 16-byte pieces, as `readable`, for elements of any size.
bool readable_rows(const at::Tensor& t) {
  const int64_t size = (int64_t)t.element_size();
  if (t.stride(3) != 1 || reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 != 0) return false;
  for (int i = 0; i < 3; ++i) {
    if (t.size(i) > INT32_MAX || (t.size(i) > 1 && t.stride(i) * size % 16 != 0)) return false;
  }
  return t.size(2) <= 1 || t.stride(2) * size < (int64_t{1} << 24);
}

// An int32 vector of n on dev that can be read as it is.
bool int32s(const at::Tensor& t, int64_t n, const c10::Device& dev) {
  return t.dim() == 1 && t.size(0) == n && t.scalar_type() == at::kInt && t.device() == dev && (n <= 1 || t.stride(0) == 1);
}

// Without the GIL from here on: an allocation or a launch may wait, and other threads of Python go on meanwhile.
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  NoGil() = default;
  NoGil(const NoGil&) = delete;
  ~NoGil() { PyEval_RestoreThread(state); }
};

bool enabled(const c10::Device& dev) {
  const int i = dev.is_cuda() ? dev.index() : -1;
  return i >= 0 && i < 64 && ((g_devices.load(std::memory_order_acquire) >> i) & 1);
}

void* stream_of(const c10::Device& dev) { return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream(); }

// The parameters that allocate_pages and release_pages share; false for operands that need preparation.
bool pages_params(const at::Tensor& table, const at::Tensor& seqlens, const at::Tensor& free_pages, const at::Tensor& num_free,
                  int64_t page_size, int64_t num_tokens, fa_pages_params& p) {
  const c10::Device dev = table.device();
  if (!enabled(dev) || table.dim() != 2 || table.scalar_type() != at::kInt) return false;
  const int64_t b = table.size(0), cols = table.size(1);
  if (b == 0 || cols == 0 || b > INT32_MAX || cols > INT32_MAX || (cols > 1 && table.stride(1) != 1) || (b > 1 && table.stride(0) < cols))
    return false;
  if (!int32s(seqlens, b, dev) || free_pages.dim() != 1 || !int32s(free_pages, free_pages.size(0), dev)) return false;
  if (num_free.numel() != 1 || num_free.scalar_type() != at::kInt || num_free.device() != dev) return false;
  if (page_size <= 0 || page_size > FA_MAX_PAGE_SIZE || num_tokens < 0 || num_tokens >= INT32_MAX || free_pages.size(0) >= INT32_MAX)
    return false;
  p.block_table = (int32_t*)table.const_data_ptr();
  p.block_table_stride = b > 1 ? table.stride(0) : 0;
  p.batch = (int32_t)b;
  p.block_table_cols = (int32_t)cols;
  p.page_size = (int32_t)page_size;
  p.free_capacity = (int32_t)free_pages.size(0);
  p.num_tokens = (int32_t)num_tokens;
  p.seqlens = (const int32_t*)seqlens.const_data_ptr();
  p.free_pages = (int32_t*)free_pages.const_data_ptr();
  p.num_free = (const int32_t*)num_free.const_data_ptr();
  return !backend_forced();
}

// (slots, cu_seqlens, seqlens, num_free), or nothing.
std::vector<at::Tensor> allocate_pages(const at::Tensor& table, const at::Tensor& seqlens, const at::Tensor& new_lens,
                                       const at::Tensor& free_pages, const at::Tensor& num_free, int64_t page_size, int64_t num_tokens) {
  fa_pages_params p{};
  if (!pages_params(table, seqlens, free_pages, num_free, page_size, num_tokens, p) || !int32s(new_lens, p.batch, table.device()))
    return {};
  const NoGil released;
  const c10::DeviceGuard guard(table.device());
  std::vector<at::Tensor> out{at::empty({num_tokens}, table.options().dtype(at::kLong)), at::empty({p.batch + 1}, table.options()),
                              at::empty({p.batch}, table.options()), at::empty(num_free.sizes(), table.options())};
  p.new_lens = (const int32_t*)new_lens.const_data_ptr();
  p.slots = (int64_t*)out[0].mutable_data_ptr();
  p.cu_seqlens = (int32_t*)out[1].mutable_data_ptr();
  p.seqlens_out = (int32_t*)out[2].mutable_data_ptr();
  p.num_free_out = (int32_t*)out[3].mutable_data_ptr();
  if (g_pages.allocate(&p, stream_of(table.device())) != FA_OK) return {};
  return out;
}

// (seqlens, num_free), or nothing.
std::vector<at::Tensor> release_pages(const at::Tensor& table, const at::Tensor& seqlens, const at::Tensor& done,
                                      const at::Tensor& free_pages, const at::Tensor& num_free, const at::Tensor& keep_lens,
                                      int64_t page_size) {
  fa_pages_params p{};
  if (!pages_params(table, seqlens, free_pages, num_free, page_size, 0, p)) return {};
  if (done.dim() != 1 || done.size(0) != p.batch || done.device() != table.device() || (p.batch > 1 && done.stride(0) != 1) ||
      (done.scalar_type() != at::kBool && done.scalar_type() != at::kByte))
    return {};
  if (keep_lens.defined() && !int32s(keep_lens, p.batch, table.device())) return {};
  const NoGil released;
  const c10::DeviceGuard guard(table.device());
  std::vector<at::Tensor> out{at::empty({p.batch}, table.options()), at::empty(num_free.sizes(), table.options())};
  p.done = (const uint8_t*)done.const_data_ptr();
  p.keep_lens = keep_lens.defined() ? (const int32_t*)keep_lens.const_data_ptr() : nullptr;
  p.seqlens_out = (int32_t*)out[0].mutable_data_ptr();
  p.num_free_out = (int32_t*)out[1].mutable_data_ptr();
  if (g_pages.release(&p, stream_of(table.device())) != FA_OK) return {};
  return out;
}

bool append_kv_paged(const at::Tensor& k, const at::Tensor& v, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& slots) {
  const c10::Device dev = k.device();
  if (!enabled(dev) || k.dim() != 3 || kc.dim() != 4 || !k.sizes().equals(v.sizes()) || !kc.sizes().equals(vc.sizes())) return false;
  if (k.scalar_type() != at::kHalf && k.scalar_type() != at::kBFloat16) return false;
  for (const at::Tensor* t : {&v, &kc, &vc}) {
    if (t->scalar_type() != k.scalar_type() || t->device() != dev) return false;
  }
  if (k.numel() == 0 || kc.numel() == 0 || k.size(2) % 8 || kc.size(1) != k.size(1) || kc.size(3) != k.size(2)) return false;
  if (slots.dim() != 1 || slots.size(0) != k.size(0) || slots.scalar_type() != at::kLong || slots.device() != dev ||
      (slots.size(0) > 1 && slots.stride(0) != 1))
    return false;
  auto in_pieces = [](const at::Tensor& t, bool written) {  // unit stride along D, whole 16 bytes
    const int64_t last = t.dim() - 1;
    if (t.stride(last) != 1 || reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 != 0) return false;
    for (int64_t i = 0; i < last; ++i) {
      if (t.size(i) > INT32_MAX || (t.size(i) > 1 && (t.stride(i) % 8 != 0 || (written && t.stride(i) <= 0)))) return false;
    }
    return true;
  };
  if (!in_pieces(k, false) || !in_pieces(v, false) || !in_pieces(kc, true) || !in_pieces(vc, true) || backend_forced()) return false;
  auto step = [](const at::Tensor& x, int i) { return x.size(i) > 1 ? x.stride(i) : 0; };
  fa_append_paged_params p{};
  p.k = k.const_data_ptr();
  p.v = v.const_data_ptr();
  p.k_stride_t = step(k, 0), p.k_stride_h = step(k, 1);
  p.v_stride_t = step(v, 0), p.v_stride_h = step(v, 1);
  p.k_cache = kc.mutable_data_ptr();
  p.v_cache = vc.mutable_data_ptr();
  p.k_page_stride = step(kc, 0), p.k_cache_stride_h = step(kc, 1), p.k_cache_stride_n = step(kc, 2);
  p.v_page_stride = step(vc, 0), p.v_cache_stride_h = step(vc, 1), p.v_cache_stride_n = step(vc, 2);
  p.slots = (const int64_t*)slots.const_data_ptr();
  p.num_tokens = (int32_t)k.size(0);
  p.heads = (int32_t)k.size(1);
  p.head_dim = (int32_t)k.size(2);
  p.num_pages = (int32_t)kc.size(0);
  p.page_size = (int32_t)kc.size(2);
  const NoGil released;
  const c10::DeviceGuard guard(dev);
  return g_pages.append(&p, stream_of(dev)) == FA_OK;
}

struct SharedCall {
  at::Tensor q, k, v, table, seqlens, prefix_lens, cu_groups, k_scale, v_scale;  // the last four may be undefined
  int64_t max_prefix, max_suffix;
  bool causal;
  double scale;
  int32_t split_len;
};

// The call's output; undefined where it needs preparation or is refused.
at::Tensor shared_prefix(const SharedCall& c) {
  const at::Tensor &q = c.q, &k = c.k, &v = c.v;
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || !q.is_cuda()) return {};
  const c10::Device dev = q.device();
  if (!enabled(dev)) return {};
  if (k.device() != dev || v.device() != dev || c.table.device() != dev) return {};
  const bool fp8 = k.scalar_type() == at::kFloat8_e4m3fn;
  if (q.scalar_type() != at::kHalf && q.scalar_type() != at::kBFloat16) return {};
  if ((!fp8 && k.scalar_type() != q.scalar_type()) || v.scalar_type() != k.scalar_type()) return {};
  if (q.numel() == 0 || k.numel() == 0 || !k.sizes().equals(v.sizes()) || k.size(3) != q.size(3) || q.size(1) % k.size(1) != 0) return {};
  const int64_t b = q.size(0), page = k.size(2);
  const at::Tensor& t = c.table;
  if (t.dim() != 2 || t.scalar_type() != at::kInt || t.size(0) != b || t.size(1) == 0 || t.size(1) > INT32_MAX ||
      (t.size(1) > 1 && t.stride(1) != 1) || (b > 1 && t.stride(0) < t.size(1)))
    return {};
  if (!int32s(c.seqlens, b, dev)) return {};
  int64_t groups = 1;
  if (c.cu_groups.defined()) {
    groups = c.cu_groups.numel() - 1;
    if (groups < 1 || groups > b || !int32s(c.cu_groups, groups + 1, dev)) return {};
  }
  if (c.prefix_lens.defined() && !int32s(c.prefix_lens, groups, dev)) return {};
  if (c.max_prefix < 0 || c.max_suffix < 0 || c.max_prefix > (1 << 29) || c.max_suffix > (1 << 29)) return {};
  if (!readable_rows(q) || !readable_rows(k) || !readable_rows(v)) return {};
  if (fp8) {
    if (page % 64 != 0 || !c.k_scale.defined() || !c.v_scale.defined()) return {};
    const int64_t want[3] = {k.size(0), k.size(1), page / 64};
    for (const at::Tensor* s : {&c.k_scale, &c.v_scale}) {
      if (s->scalar_type() != at::kFloat || s->device() != dev || !s->sizes().equals(at::IntArrayRef(want, 3)) || s->stride(2) != 1)
        return {};
    }
    if (!c.k_scale.strides().equals(c.v_scale.strides())) return {};
  }
  if (backend_forced()) return {};

  const NoGil released;
  const c10::DeviceGuard guard(dev);
  at::Tensor o = at::empty(q.sizes(), q.options());
  auto step = [](const at::Tensor& x, int i) { return x.size(i) > 1 ? x.stride(i) : 0; };
  fa_fwd_params p{};
  p.q = q.const_data_ptr();
  p.k = k.const_data_ptr();
  p.v = v.const_data_ptr();
  p.o = o.mutable_data_ptr();
  p.q_stride_b = step(q, 0), p.q_stride_h = step(q, 1), p.q_stride_n = step(q, 2);
  p.k_stride_h = step(k, 1), p.k_stride_n = step(k, 2);
  p.v_stride_h = step(v, 1), p.v_stride_n = step(v, 2);
  p.o_stride_b = step(o, 0), p.o_stride_h = step(o, 1), p.o_stride_n = step(o, 2);
  p.batch = (int32_t)b;
  p.heads_q = (int32_t)q.size(1);
  p.heads_kv = (int32_t)k.size(1);
  p.seqlen_q = (int32_t)q.size(2);
  p.head_dim = (int32_t)q.size(3);
  p.scale = (float)c.scale;
  p.causal = c.causal ? 1 : 0;
  p.dtype = dtype_code(q.scalar_type());
  p.kv_dtype = fp8 ? FA_DTYPE_FP8_E4M3 : p.dtype;
  if (fp8) {
    p.k_scale = (const float*)c.k_scale.const_data_ptr();
    p.v_scale = (const float*)c.v_scale.const_data_ptr();
    p.scale_stride_b = c.k_scale.stride(0);
    p.scale_stride_h = c.k_scale.stride(1);
  }
  fa_paged_kv kv{};
  kv.block_table = (const int32_t*)t.const_data_ptr();
  kv.block_table_stride = t.stride(0);
  kv.block_table_cols = (int32_t)t.size(1);
  kv.page_size = (int32_t)page;
  kv.seqlens_k = (const int32_t*)c.seqlens.const_data_ptr();
  kv.num_pages = (int32_t)k.size(0);
  kv.k_page_stride = step(k, 0);
  kv.v_page_stride = step(v, 0);
  fa_shared_prefix s{};
  s.prefix_lens = c.prefix_lens.defined() ? (const int32_t*)c.prefix_lens.const_data_ptr() : nullptr;
  s.cu_groups = c.cu_groups.defined() ? (const int32_t*)c.cu_groups.const_data_ptr() : nullptr;
  s.num_groups = (int32_t)groups;
  s.max_prefix_len = (int32_t)c.max_prefix;
  s.max_suffix_len = (int32_t)c.max_suffix;
  s.split_len = c.split_len;
  const size_t need = g_shared.workspace_bytes(&p, &kv, &s);
  if (need == 0) return {};  // refused: the Python code reports it
  const at::Tensor ws = at::empty({(int64_t)(need / 4)}, q.options().dtype(at::kFloat));
  return g_shared.call(&p, &kv, &s, ws.mutable_data_ptr(), need, stream_of(dev)) == FA_OK ? o : at::Tensor();
}

// What f makes of tensors (those in `maybe` may be None), or None.  Nothing is thrown and no Python error is left: what
// fails here (memory, say) fails again in the Python code, which reports it.
template <class F>
PyObject* with_tensors(std::initializer_list<PyObject*> always, std::initializer_list<PyObject*> maybe, F&& f) {
  try {
    for (PyObject* o : always) {
      if (!THPVariable_CheckExact(o)) Py_RETURN_NONE;
    }
    for (PyObject* o : maybe) {
      if (o != Py_None && !THPVariable_CheckExact(o)) Py_RETURN_NONE;
    }
    if (PyObject* out = f()) return out;
  } catch (const std::exception&) {
  }
  PyErr_Clear();
  Py_RETURN_NONE;
}

at::Tensor tensor_or_none(PyObject* o) { return o == Py_None ? at::Tensor() : THPVariable_Unpack(o); }

PyObject* tuple_of(const std::vector<at::Tensor>& out) {
  PyObject* t = out.empty() ? nullptr : PyTuple_New((Py_ssize_t)out.size());
  for (size_t i = 0; t != nullptr && i < out.size(); ++i) {
    PyObject* o = THPVariable_Wrap(out[i]);
    if (o == nullptr) {
      Py_DECREF(t);
      return nullptr;
    }
    PyTuple_SET_ITEM(t, (Py_ssize_t)i, o);
  }
  return t;
}

// Numbers among the arguments: anything else, or past the range, ends the call (as above: None).
struct NoNumber : std::exception {};
int64_t whole(PyObject* o) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred() != nullptr) throw NoNumber();
  return x;
}
int32_t whole32(PyObject* o) {
  const int64_t x = whole(o);
  if (x < INT32_MIN || x > INT32_MAX) throw NoNumber();
  return (int32_t)x;
}
double real(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred() != nullptr) throw NoNumber();
  return x;
}

bool takes(Py_ssize_t given, Py_ssize_t wanted) {
  if (given != wanted) PyErr_Format(PyExc_TypeError, "%zd arguments in place of %zd", given, wanted);
  return given == wanted;
}

// attention_shared_prefix of (q, k, v, block_table, seqlens_k, prefix_lens or None, cu_groups or None, k_scale or None, v_scale
// or None, max_prefix, max_suffix, causal, scale, split_len or 0): its output.
PyObject* py_shared_prefix(PyObject*, PyObject* const* x, Py_ssize_t n) {
  if (!takes(n, 14)) return nullptr;
  return with_tensors({x[0], x[1], x[2], x[3], x[4]}, {x[5], x[6], x[7], x[8]}, [&]() -> PyObject* {
    const at::Tensor out = shared_prefix({THPVariable_Unpack(x[0]), THPVariable_Unpack(x[1]), THPVariable_Unpack(x[2]),
                                          THPVariable_Unpack(x[3]), THPVariable_Unpack(x[4]), tensor_or_none(x[5]),
                                          tensor_or_none(x[6]), tensor_or_none(x[7]), tensor_or_none(x[8]), whole(x[9]), whole(x[10]),
                                          whole(x[11]) != 0, real(x[12]), whole32(x[13])});
    return out.defined() ? THPVariable_Wrap(out) : nullptr;
  });
}

// allocate_pages of (block_table, seqlens_k, new_lens, free_pages, num_free, page_size, num_tokens): a tuple.
PyObject* py_allocate_pages(PyObject*, PyObject* const* x, Py_ssize_t n) {
  if (!takes(n, 7)) return nullptr;
  return with_tensors({x[0], x[1], x[2], x[3], x[4]}, {}, [&] {
    return tuple_of(allocate_pages(THPVariable_Unpack(x[0]), THPVariable_Unpack(x[1]), THPVariable_Unpack(x[2]),
                                   THPVariable_Unpack(x[3]), THPVariable_Unpack(x[4]), whole(x[5]), whole(x[6])));
  });
}

// release_pages of (block_table, seqlens_k, done, free_pages, num_free, keep_lens or None, page_size): a tuple.
PyObject* py_release_pages(PyObject*, PyObject* const* x, Py_ssize_t n) {
  if (!takes(n, 7)) return nullptr;
  return with_tensors({x[0], x[1], x[2], x[3], x[4]}, {x[5]}, [&] {
    return tuple_of(release_pages(THPVariable_Unpack(x[0]), THPVariable_Unpack(x[1]), THPVariable_Unpack(x[2]),
                                  THPVariable_Unpack(x[3]), THPVariable_Unpack(x[4]), tensor_or_none(x[5]), whole(x[6])));
  });
}

// append_kv_paged of (k, v, k_cache, v_cache, slots): True.
PyObject* py_append_kv_paged(PyObject*, PyObject* const* x, Py_ssize_t n) {
  if (!takes(n, 5)) return nullptr;
  return with_tensors({x[0], x[1], x[2], x[3], x[4]}, {}, [&]() -> PyObject* {
    if (!append_kv_paged(THPVariable_Unpack(x[0]), THPVariable_Unpack(x[1]), THPVariable_Unpack(x[2]), THPVariable_Unpack(x[3]),
                         THPVariable_Unpack(x[4])))
      return nullptr;
    Py_RETURN_TRUE;
  });
}

// (functions of Python's own calling convention: through ctypes a call took 0.2 to 0.6 us more)
template <class F>
PyCFunction function(F* f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}
PyMethodDef kFunctions[] = {{"shared_prefix", function(py_shared_prefix), METH_FASTCALL, nullptr},
                            {"allocate_pages", function(py_allocate_pages), METH_FASTCALL, nullptr},
                            {"release_pages", function(py_release_pages), METH_FASTCALL, nullptr},
                            {"append_kv_paged", function(py_append_kv_paged), METH_FASTCALL, nullptr},
                            {nullptr, nullptr, 0, nullptr}};

// Autograd: the op has no formula of its own, so a call that would record one goes to the Python kernel, which
// records the node that the op's users registered, or one that raises.
at::Tensor attention_autograd(c10::DispatchKeySet ks, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool causal,
                              std::optional<double> scale) {
  if (c10::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return call_python(c10::DispatchKey::Autograd, q, k, v, causal, scale);
  using Fn = at::Tensor(const at::Tensor&, const at::Tensor&, const at::Tensor&, bool, std::optional<double>);
  static const auto op = attention_op().typed<Fn>();
  const at::AutoDispatchBelowAutograd below;
  return op.redispatch(ks & c10::after_autograd_keyset, q, k, v, causal, scale);
}

}  // namespace

extern "C" {

// What this library was built against: a torch build has no stable C++ ABI, and the HIP library bound below may come
// from elsewhere.  Python compares them before it registers the kernels, so loading the library has no effect.
const char* fa_torch_built_for(void) { return FA_TORCH_BUILD; }
int32_t fa_torch_abi_version(void) { return FA_ABI_VERSION; }
size_t fa_torch_params_size(void) { return sizeof(fa_fwd_params); }

// Registers the kernels, once; 0 when torch refuses them.
int32_t fa_torch_register(void) {
  try {
    static torch::Library cuda(torch::Library::IMPL, "fused_attn", c10::DispatchKey::CUDA, __FILE__, __LINE__);
    static torch::Library autograd(torch::Library::IMPL, "fused_attn", c10::DispatchKey::AutogradCUDA, __FILE__, __LINE__);
    static const bool once = (cuda.impl("attention", TORCH_FN(attention_gpu)), autograd.impl("attention", TORCH_FN(attention_autograd)), true);
    return once;
  } catch (const std::exception&) {
    return 0;
  }
}

void fa_torch_bind(void* fwd_workspace_bytes, void* fwd_ws, void* splitk_workspace_bytes, void* splitk, void* last_error) {
  g_abi.fwd_workspace_bytes = (decltype(g_abi.fwd_workspace_bytes))fwd_workspace_bytes;
  g_abi.fwd_ws = (decltype(g_abi.fwd_ws))fwd_ws;
  g_abi.splitk_workspace_bytes = (decltype(g_abi.splitk_workspace_bytes))splitk_workspace_bytes;
  g_abi.splitk = (decltype(g_abi.splitk))splitk;
  g_abi.last_error = (decltype(g_abi.last_error))last_error;
}

void fa_torch_bind_shared(void* workspace_bytes, void* call) {
  g_shared.workspace_bytes = (decltype(g_shared.workspace_bytes))workspace_bytes;
  g_shared.call = (decltype(g_shared.call))call;
}

void fa_torch_bind_pages(void* allocate, void* release, void* append) {
  g_pages.allocate = (decltype(g_pages.allocate))allocate;
  g_pages.release = (decltype(g_pages.release))release;
  g_pages.append = (decltype(g_pages.append))append;
}

// {name: function} of the Python functions above, called with the GIL held.
PyObject* fa_torch_functions(void) {
  PyObject* all = PyDict_New();
  for (PyMethodDef* m = kFunctions; all != nullptr && m->ml_name != nullptr; ++m) {
    PyObject* f = PyCFunction_New(m, nullptr);
    const bool kept = f != nullptr && PyDict_SetItemString(all, m->ml_name, f) == 0;
    Py_XDECREF(f);
    if (!kept) Py_CLEAR(all);
  }
  return all;
}

// Device `index` runs the library bound above (which happens before).
void fa_torch_enable(int32_t index) {
  if (index >= 0 && index < 64) g_devices.fetch_or(uint64_t{1} << index, std::memory_order_release);
}

int32_t fa_torch_backend_forced(void) { return backend_forced(); }

int64_t fa_torch_route(int32_t half, int64_t b, int64_t hq, int64_t hkv, int64_t nq, int64_t nk, int64_t d) {
  return route(half != 0, b, hq, hkv, nq, nk, d);
}

}  // extern "C"
