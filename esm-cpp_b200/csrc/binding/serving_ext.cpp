// Python binding of the token-by-token serving operators: the checks of the
// tensors, the outputs and workspaces (torch's allocator), torch's current
// stream, and one call of the C ABI.  A decoding step makes many of these
// calls, each a few microseconds of device time; read from Python, the nine
// tensors of an append cost more host time than their checks and the launch
// take here.
//
// The library itself stays free of torch: this module is handed the addresses
// of its functions (bind) and passes plain pointers.  The GIL is held from the
// binding of the stream to the return, so that threads on streams of their own
// can call at once although they share one context per device.
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <cstdint>
#include <map>
#include <optional>
#include <string>
#include <type_traits>

#include "esm_b200.h"

namespace {

using at::Tensor;

struct Library {
  decltype(&esmcu_open) open = nullptr;
  decltype(&esmcu_set_stream) set_stream = nullptr;
  decltype(&esmcu_synchronize) synchronize = nullptr;
  decltype(&esmcu_linear_w4) linear_w4 = nullptr;
  decltype(&esmcu_linear_w4_workspace) linear_w4_workspace = nullptr;
  decltype(&esmcu_kv_append_paged) kv_append_paged = nullptr;
  decltype(&esmcu_attention_decode_paged) attention_decode_paged = nullptr;
  decltype(&esmcu_attention_decode_paged_workspace) attention_decode_paged_workspace = nullptr;
  py::object check;  // _lib.check: raises for a status that is not OK
};
// Never destroyed: it holds a Python object, and module-level destructors run
// after the interpreter.
Library& lib() {
  static Library* l = new Library();
  return *l;
}

void check(int rc, const char* name) {
  if (rc != ESMCU_OK) lib().check(rc, name);
}

// One context per device, apart from the facade's, and the stream that it is
// bound to.
struct Context {
  esmcu_context* handle = nullptr;
  void* stream = nullptr;
};
std::map<int, Context>& contexts() {
  static auto* m = new std::map<int, Context>();
  return *m;
}

// `device` current, its context bound to torch's current stream; the current
// device is put back at the end.
class Bound {
 public:
  explicit Bound(int device) : before_(c10::cuda::current_device()), device_(device) {
    if (before_ != device_) c10::cuda::set_device(device_);
    try {
      Context& c = contexts()[device_];
      if (c.handle == nullptr) check(lib().open(device_, &c.handle), "esmcu_open");
      void* s = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device_)).stream();
      if (s == nullptr) s = reinterpret_cast<void*>(1);  // cudaStreamLegacy; NULL would be the context's own
      if (s != c.stream) {
        check(lib().set_stream(c.handle, s), "esmcu_set_stream");
        c.stream = s;
      }
      handle_ = c.handle;
    } catch (...) {
      restore();
      throw;
    }
  }
  ~Bound() { restore(); }
  esmcu_context* get() const { return handle_; }

 private:
  void restore() noexcept {
    try {
      if (before_ != device_) c10::cuda::set_device(before_);
    } catch (...) {
    }
  }
  int before_, device_;
  esmcu_context* handle_ = nullptr;
};

#define NEED(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

int code_of(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return ESMCU_F32;
    case at::kHalf: return ESMCU_F16;
    case at::kBFloat16: return ESMCU_BF16;
    default: NEED(false, what, " must be float32, float16 or bfloat16"); return -1;
  }
}

bool last_contiguous(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }

// The stride of a dimension; torch may give one of a single entry any stride.
int64_t step(const Tensor& t, int64_t dim, int64_t single = 0) { return t.size(dim) > 1 ? t.stride(dim) : single; }

int as_int(int64_t v, const char* what) {
  NEED(v >= 0 && v <= INT32_MAX, what, " is out of range");
  return static_cast<int>(v);
}

bool same_device(const Tensor& t, const Tensor& as) { return t.device() == as.device(); }

// These operators have no backward pass; an output without the gradient that a
// caller expects would say nothing.
template <typename... T>
void refuse_gradients(const T&... tensors) {
  auto wants = [](const auto& t) {
    if constexpr (std::is_same_v<std::decay_t<decltype(t)>, Tensor>) return t.requires_grad();
    else return t.has_value() && t->requires_grad();
  };
  NEED(!at::GradMode::is_enabled() || !(wants(tensors) || ...),
       "an input requires a gradient, and the serving operators have no backward pass: call them under "
       "torch.no_grad(), or detach it");
}

// Counts a write that autograd has to know of: a tensor that a graph keeps for its
// backward pass is then refused there.
void count_write(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A workspace on the current device, in the order of its current stream; back
// with torch's allocator (a captured call's graph keeps it) when it goes.
c10::DataPtr workspace(size_t bytes) { return c10::cuda::CUDACachingAllocator::get()->allocate(bytes); }

Tensor linear_w4(const Tensor& x, const Tensor& wq, const Tensor& scales, const std::optional<Tensor>& zeros,
                 const std::optional<Tensor>& bias, int64_t group_size) {
  refuse_gradients(x, scales, bias);
  NEED(x.dim() == 2 && wq.dim() == 2 && scales.dim() == 2, "x, wq and scales must be matrices");
  NEED(x.is_cuda(), "x must be a CUDA tensor");
  const int64_t M = x.size(0), K = x.size(1), N = wq.size(0), half = (K + 1) / 2;
  esmcu_linear_w4_args a = {};
  a.dtype = code_of(x, "x");
  a.scales_dtype = code_of(scales, "scales");
  NEED(group_size == 32 || group_size == 64 || group_size == 128, "group_size must be 32, 64 or 128");
  const int64_t groups = (K + group_size - 1) / group_size;
  NEED(wq.scalar_type() == at::kByte && wq.size(1) == half, "wq must be uint8 [N, ", half, "] for K = ", K);
  NEED(scales.size(0) == N && scales.size(1) == groups, "scales must be [", N, ", ", groups, "]");
  NEED(same_device(wq, x) && same_device(scales, x), "wq and scales must be on x's device");
  NEED(last_contiguous(x) && last_contiguous(wq) && last_contiguous(scales),
       "x, wq and scales must be contiguous in their last dimension");
  if (zeros) {
    NEED(zeros->sizes() == scales.sizes() && zeros->scalar_type() == at::kByte && same_device(*zeros, x),
         "zeros must be uint8, of the shape and on the device of scales");
    NEED(last_contiguous(*zeros), "zeros must be contiguous in its last dimension");
    a.zeros = zeros->const_data_ptr<uint8_t>();
    a.ldz = step(*zeros, 0, groups);
  }
  if (bias) {
    NEED(bias->dim() == 1 && bias->size(0) == N && bias->scalar_type() == at::kFloat && same_device(*bias, x) &&
             bias->is_contiguous(),
         "bias must be contiguous float32 [", N, "] on x's device");
    a.bias = bias->const_data_ptr<float>();
  }
  a.M = as_int(M, "M");
  a.N = as_int(N, "N");
  a.K = as_int(K, "K");
  a.group = static_cast<int>(group_size);
  a.x = x.const_data_ptr();
  a.ldx = step(x, 0, K);
  a.wq = wq.const_data_ptr<uint8_t>();
  a.ldw = step(wq, 0, half);
  a.scales = scales.const_data_ptr();
  a.lds = step(scales, 0, groups);
  Tensor out = at::empty({M, N}, x.options());
  a.out = out.mutable_data_ptr();
  a.ldo = N;
  check(lib().linear_w4_workspace(a.dtype, a.M, a.K, a.group, &a.workspace_bytes), "esmcu_linear_w4_workspace");
  Bound ctx(x.get_device());
  c10::DataPtr work;
  if (a.workspace_bytes > 0) {
    work = workspace(a.workspace_bytes);
    a.workspace = work.get();
  }
  check(lib().linear_w4(ctx.get(), &a), "esmcu_linear_w4");
  return out;
}

esmcu_paged_kv paged(const Tensor& k, const Tensor& v, const Tensor& table, int64_t sequences) {
  NEED(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(),
       "k_cache and v_cache must be [pages, page_size, kv_heads, head_dim], of one shape and type");
  NEED(k.is_cuda(), "k_cache must be a CUDA tensor");
  esmcu_paged_kv c = {};
  c.dtype = code_of(k, "the cache");
  NEED(table.dim() == 2 && table.scalar_type() == at::kInt && table.size(0) >= sequences,
       "page_table must be int32 [sequences, max_pages] for at least ", sequences, " sequences");
  NEED(same_device(v, k) && same_device(table, k), "k_cache, v_cache and page_table must be on one device");
  NEED(last_contiguous(k) && last_contiguous(v) && last_contiguous(table),
       "k_cache, v_cache and page_table must be contiguous in their last dimension");
  c.k = k.mutable_data_ptr();
  c.v = v.mutable_data_ptr();
  c.num_pages = as_int(k.size(0), "pages");
  c.page_size = as_int(k.size(1), "page_size");
  c.num_kv_heads = as_int(k.size(2), "kv_heads");
  c.head_dim = as_int(k.size(3), "head_dim");
  c.k_stride_page = step(k, 0);
  c.k_stride_slot = step(k, 1);
  c.k_stride_head = step(k, 2);
  c.v_stride_page = step(v, 0);
  c.v_stride_slot = step(v, 1);
  c.v_stride_head = step(v, 2);
  c.page_table = table.const_data_ptr<int32_t>();
  c.page_table_stride = step(table, 0);
  c.max_pages = as_int(table.size(1), "max_pages");
  return c;
}

bool int_vector(const Tensor& t, int64_t n, const Tensor& as) {
  return t.dim() == 1 && t.size(0) == n && t.scalar_type() == at::kInt && t.is_contiguous() && same_device(t, as);
}

std::optional<Tensor> kv_append_paged(const Tensor& k, const Tensor& v, const Tensor& k_cache, const Tensor& v_cache,
                                      const Tensor& page_table, const Tensor& cu_seqlens, const Tensor& cache_lens,
                                      const std::optional<Tensor>& q, const std::optional<Tensor>& cos,
                                      const std::optional<Tensor>& sin) {
  refuse_gradients(k, v, k_cache, v_cache, q, cos, sin);
  NEED(cache_lens.dim() == 1, "cache_lens must be [B]");
  const int64_t B = cache_lens.size(0);
  const esmcu_paged_kv cache = paged(k_cache, v_cache, page_table, B);
  NEED(k.dim() == 3 && k.size(1) == cache.num_kv_heads && k.size(2) == cache.head_dim && v.sizes() == k.sizes(),
       "k and v must be [T, kv_heads, head_dim] with the cache's heads");
  NEED((k.scalar_type() == k_cache.scalar_type() || k.scalar_type() == at::kFloat) && v.scalar_type() == k.scalar_type(),
       "k and v must have the cache's type or be float32, both the same");
  NEED(int_vector(cu_seqlens, B + 1, k_cache) && int_vector(cache_lens, B, k_cache),
       "cu_seqlens [B + 1] and cache_lens [B] must be contiguous int32 on the cache's device");
  NEED(same_device(k, k_cache) && same_device(v, k_cache), "k and v must be on the cache's device");
  NEED(last_contiguous(k) && last_contiguous(v), "k and v must be contiguous in their last dimension");
  const int64_t T = k.size(0);
  esmcu_kv_append_args a = {};
  a.dtype = code_of(k, "k");
  a.k = k.const_data_ptr();
  a.v = v.const_data_ptr();
  a.k_stride_token = step(k, 0);
  a.k_stride_head = step(k, 1);
  a.v_stride_token = step(v, 0);
  a.v_stride_head = step(v, 1);
  a.cu_seqlens = cu_seqlens.const_data_ptr<int32_t>();
  a.cache_lens = cache_lens.const_data_ptr<int32_t>();
  a.B = as_int(B, "B");
  a.T = as_int(T, "T");
  std::optional<Tensor> out;
  if (q) {
    NEED(q->dim() == 3 && q->size(0) == T && q->size(2) == cache.head_dim && q->scalar_type() == k.scalar_type() &&
             same_device(*q, k_cache),
         "q must be [T, q_heads, head_dim] of k's type, on the cache's device");
    NEED(last_contiguous(*q), "q must be contiguous in its last dimension");
    out = at::empty({T, q->size(1), cache.head_dim}, k_cache.options());
    a.num_q_heads = as_int(q->size(1), "q_heads");
    if (a.num_q_heads > 0) {
      a.q = q->const_data_ptr();
      a.q_out = out->mutable_data_ptr();
      a.q_stride_token = step(*q, 0);
      a.q_stride_head = step(*q, 1);
    }
  }
  if (cos || sin) {
    NEED(cos && sin && cos->dim() == 2 && sin->sizes() == cos->sizes(), "cos and sin must both be [positions, rot]");
    NEED(cos->scalar_type() == at::kFloat && sin->scalar_type() == at::kFloat && cos->is_contiguous() &&
             sin->is_contiguous() && same_device(*cos, k_cache) && same_device(*sin, k_cache),
         "cos and sin must be contiguous float32 on the cache's device");
    a.table_rows = as_int(cos->size(0), "positions");
    a.rot_dim = as_int(cos->size(1), "rot");
    a.cos_t = cos->const_data_ptr<float>();
    a.sin_t = sin->const_data_ptr<float>();
  }
  if (T > 0 && B > 0) {
    Bound ctx(k_cache.get_device());
    check(lib().kv_append_paged(ctx.get(), &cache, &a), "esmcu_kv_append_paged");
    count_write(k_cache);
    count_write(v_cache);
  }
  return out;
}

py::object attention_decode_paged(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& page_table,
                                  const Tensor& seq_lens, double scale, int64_t window, bool return_lse) {
  refuse_gradients(q, k_cache, v_cache);
  NEED(q.dim() == 3, "q must be [B, q_heads, head_dim]");
  const int64_t B = q.size(0);
  const esmcu_paged_kv cache = paged(k_cache, v_cache, page_table, B);
  NEED(q.size(2) == cache.head_dim && q.scalar_type() == k_cache.scalar_type(),
       "q must have the cache's head_dim and type");
  NEED(same_device(q, k_cache) && int_vector(seq_lens, B, k_cache),
       "q and contiguous int32 seq_lens [", B, "] must be on the cache's device");
  NEED(last_contiguous(q), "q must be contiguous in its last dimension");
  esmcu_attention_decode_args a = {};
  a.q = q.const_data_ptr();
  a.q_stride_seq = step(q, 0);
  a.q_stride_head = step(q, 1);
  a.num_q_heads = as_int(q.size(1), "q_heads");
  a.B = as_int(B, "B");
  a.seq_lens = seq_lens.const_data_ptr<int32_t>();
  a.scale = static_cast<float>(scale);
  a.window = window > INT32_MAX ? INT32_MAX : window < 0 ? -1 : static_cast<int>(window);
  Bound ctx(k_cache.get_device());
  check(lib().attention_decode_paged_workspace(ctx.get(), &cache, a.num_q_heads, &a.workspace_bytes),
        "esmcu_attention_decode_paged_workspace");
  Tensor out = at::empty(q.sizes(), q.options());
  Tensor lse;
  const c10::DataPtr work = workspace(a.workspace_bytes);
  a.out = out.mutable_data_ptr();
  a.workspace = work.get();
  if (return_lse) {
    lse = at::empty({B, q.size(1)}, q.options().dtype(at::kFloat));
    a.lse = lse.mutable_data_ptr<float>();
  }
  check(lib().attention_decode_paged(ctx.get(), &cache, &a), "esmcu_attention_decode_paged");
  if (return_lse) return py::make_tuple(out, lse);
  return py::cast(out);
}

// Reports what the device found wrong since the last report; the caller has
// waited for the stream.
void synchronize(int device) {
  if (contexts().count(device) == 0 || contexts()[device].handle == nullptr) return;
  Bound ctx(device);
  check(lib().synchronize(ctx.get()), "esmcu_synchronize");
}

template <typename F>
void set(F& f, const py::dict& addresses, const char* name) {
  f = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

void bind(const py::dict& addresses, py::object check) {
  Library& l = lib();
  set(l.open, addresses, "esmcu_open");
  set(l.set_stream, addresses, "esmcu_set_stream");
  set(l.synchronize, addresses, "esmcu_synchronize");
  set(l.linear_w4, addresses, "esmcu_linear_w4");
  set(l.linear_w4_workspace, addresses, "esmcu_linear_w4_workspace");
  set(l.kv_append_paged, addresses, "esmcu_kv_append_paged");
  set(l.attention_decode_paged, addresses, "esmcu_attention_decode_paged");
  set(l.attention_decode_paged_workspace, addresses, "esmcu_attention_decode_paged_workspace");
  l.check = std::move(check);
}

}  // namespace

PYBIND11_MODULE(_serving_ext, m) {
  m.def("bind", &bind, py::arg("addresses"), py::arg("check"));
  m.def("synchronize", &synchronize, py::arg("device"));
  m.def("linear_w4", &linear_w4, py::arg("x"), py::arg("wq"), py::arg("scales"), py::arg("zeros") = py::none(),
        py::arg("bias") = py::none(), py::arg("group_size") = 128, R"(
A Linear with 4-bit weights and group scales, for few rows:
out[m, n] = sum_k x[m, k] * (q[n, k] - z[n, k // group_size])
* scales[n, k // group_size] + bias[n], of x's type.

x [M, K] float32, float16 or bfloat16; wq uint8 [N, ceil(K / 2)], column 2j
in the low four bits of byte j; scales [N, ceil(K / group_size)] of any of
the three types; zeros uint8 of the same shape with values 0 to 15 (None: 8
everywhere); bias float32 [N]; group_size 32, 64 or 128
(prep.quantize_weight_w4 makes wq and scales); K at most 131072.  Sums are
float32, rounded once; in 16-bit x an element some thousands of times above its
256 columns costs the others bits, also where its weight is 0.  Rows of wq that start on 16-byte boundaries are read
fastest.  No backward pass: inputs that require gradients are refused unless
gradients are off.)");
  m.def("kv_append_paged", &kv_append_paged, py::arg("k"), py::arg("v"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("page_table"), py::arg("cu_seqlens"), py::arg("cache_lens"), py::arg("q") = py::none(),
        py::arg("cos") = py::none(), py::arg("sin") = py::none(), R"(
Appends packed new tokens to a paged K/V cache, RoPE applied on the way;
returns the rotated queries (None without q).

k, v [T, kv_heads, dh] and q [T, q_heads, dh] in the cache's type, or
float32 to be rounded to it (views into a joint qkv row are fine); k_cache
and v_cache [pages, page_size, kv_heads, dh], any strides with contiguous
heads' elements, written in place; page_table int32 [B, max_pages];
cu_seqlens int32 [B + 1]; cache_lens int32 [B], the tokens already cached
(not advanced).  Token t of sequence b goes to position
cache_lens[b] + t - cu_seqlens[b].  cos and sin float32 [positions, rot]
rotate the first rot (<= dh) elements of every q and k head by the row of
the token's position, as rope_build_tables lays them out; None: no
rotation.  Rows behind cu_seqlens[B] are left out (their q rows hold
nothing).  A position or page id outside the cache or the tables is
skipped and reported by synchronize().  No backward pass: inputs that require
gradients are refused unless gradients are off.)");
  m.def("attention_decode_paged", &attention_decode_paged, py::arg("q"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("page_table"), py::arg("seq_lens"), py::arg("scale") = 1.0, py::arg("window") = 0,
        py::arg("return_lse") = false, R"(
Attention of one new token per sequence over a paged K/V cache:
out[b, h] = sum_t softmax_t(scale * q[b, h] . k[t, h']) v[t, h'] over the
seq_lens[b] cached keys (the last `window` of them when window > 0),
h' = h // (q_heads // kv_heads).

q [B, q_heads, dh] of the cache's type (pre-scaled for scale = 1, as for
attention_varlen); caches and page_table as for kv_append_paged, dh a
multiple of 8 up to 256 and rows on 16-byte boundaries; seq_lens int32 [B],
on the device, the new token's own key included.  Returns out [B, q_heads,
dh], and with return_lse also float32 log(sum_t exp(scale * q . k))
[B, q_heads].  A sequence of length 0 gives zeros and -inf; an infinite
element of a seen v row gives NaN or an infinity.  A length or
page id outside the cache is skipped and reported by synchronize().  No
backward pass: inputs that require gradients are refused unless gradients are
off.)");
}
