// Host path of the serving operators (serving.py): argument checks, output
// allocation and the call into the C ABI, in C++.
//
// A decode step calls these operators a few times per layer with kernels of
// 2 to 12 us; through ctypes and torch's Python allocation calls a call cost 10
// to 20 us of host time, here about 6.  Nothing is computed here and nothing is kept between calls:
// the C entry points (include/bsgemm.h) do the work and check what they are
// given again.  Their addresses come from the library that _lib.py loaded, so
// there is one copy of it.
#include <ATen/MemoryOverlap.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/types.h>

#include <optional>
#include <string>

#include "../../include/bsgemm.h"

namespace py = pybind11;
using Opt = std::optional<at::Tensor>;

namespace {

decltype(&bs_rms_norm) p_rms_norm;
decltype(&bs_rms_norm_quant) p_rms_norm_quant;
decltype(&bs_rope) p_rope;
decltype(&bs_cache_append) p_cache_append;
decltype(&bs_cache_attn) p_cache_attn;
decltype(&bs_cache_attn_workspace_size) p_cache_attn_ws;

void bind(const py::dict& address) {
  auto get = [&](const char* name, auto& fn) {
    fn = reinterpret_cast<std::decay_t<decltype(fn)>>(address[name].cast<uintptr_t>());
  };
  get("bs_rms_norm", p_rms_norm);
  get("bs_rms_norm_quant", p_rms_norm_quant);
  get("bs_rope", p_rope);
  get("bs_cache_append", p_cache_append);
  get("bs_cache_attn", p_cache_attn);
  get("bs_cache_attn_workspace_size", p_cache_attn_ws);
}

// Messages are put together without iostreams: formatting a number through one crashed here (facets of another copy of
// the C++ library in the process).
std::string str(const char* s) { return s; }
std::string str(int64_t v) { return std::to_string(v); }
std::string str(at::ScalarType t) { return c10::toString(t); }
std::string str(const c10::Device& d) { return d.str(); }
std::string str(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}
template <class... A>
std::string text(const A&... a) {
  return (std::string() + ... + str(a));
}
template <class... A>
[[noreturn]] void bad_type(const A&... a) { throw py::type_error(text(a...)); }
template <class... A>
[[noreturn]] void bad_value(const A&... a) { throw py::value_error(text(a...)); }

const void* ptr(const Opt& t) { return t ? t->const_data_ptr() : nullptr; }

int tag(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return BS_DT_F32;
    case at::kBFloat16: return BS_DT_BF16;
    case at::kHalf: return BS_DT_F16;
    default: return -1;
  }
}

// The device that all tensors are on, current while this lives; its current stream.
struct On {
  c10::DeviceIndex index;
  c10::cuda::OptionalCUDAGuard guard;
  void* stream;
  template <class... T>
  explicit On(const at::Tensor& first, const T&... rest) {
    if (!first.is_cuda()) throw std::runtime_error("bsgemm ops run on CUDA tensors only (no CPU fallback)");
    index = first.get_device();
    (same(first, rest), ...);
    if (c10::cuda::current_device() != index) guard.set_index(index);
    stream = c10::cuda::getCurrentCUDAStream(index).stream();
  }
  static void same(const at::Tensor& a, const at::Tensor& b) {
    if (!b.is_cuda() || a.get_device() != b.get_device()) bad_value("tensors on ", a.device(), " and ", b.device());
  }
  static void same(const at::Tensor& a, const Opt& b) {
    if (b) same(a, *b);
  }
};

at::Tensor empty(const at::Tensor& like, at::IntArrayRef shape, at::ScalarType dtype) {
  return at::empty(shape, like.options().dtype(dtype).memory_format(at::MemoryFormat::Contiguous));
}

bool misaligned(const at::Tensor& t, uintptr_t a) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % a != 0; }

// What torch's own in-place operators do: autograd's saved tensors then notice that their values are gone.
void changed(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// t, or a copy where it is not contiguous or does not start on 16 bytes.
at::Tensor dense(const at::Tensor& t) {
  return t.is_contiguous() && !misaligned(t, 16) ? t : t.clone(at::MemoryFormat::Contiguous);
}

// Status and outputs; the caller turns a status into its exception.
py::tuple rms(const at::Tensor& x, const at::Tensor& weight, double eps, const Opt& residual, bool codes, bool pow2, bool e8m0) {
  const On on(x, weight, residual);
  const auto dt = x.scalar_type();
  if (tag(dt) < 0) bad_type("rms_norm: x is ", dt, ", expected bf16, f16 or fp32");
  if (weight.scalar_type() != dt || (residual && residual->scalar_type() != dt))
    bad_type("rms_norm: x, weight and residual must have one type");
  if (x.dim() < 1 || weight.dim() != 1 || weight.size(0) != x.size(-1))
    bad_value("rms_norm: weight ", weight.sizes(), " does not match x ", x.sizes());
  if (residual && residual->sizes() != x.sizes()) bad_value("rms_norm: residual ", residual->sizes(), " does not match x ", x.sizes());
  const int64_t H = x.size(-1);
  const at::Tensor xc = dense(x), wc = dense(weight), rc = residual ? dense(*residual) : at::Tensor();
  at::Tensor h = residual ? empty(x, x.sizes(), dt) : at::Tensor();
  const int64_t rows = H ? x.numel() / H : 0;
  const void* r = residual ? rc.const_data_ptr() : nullptr;
  void* hp = residual ? h.mutable_data_ptr() : nullptr;
  if (!codes) {
    at::Tensor y = empty(x, x.sizes(), dt);
    const int st = p_rms_norm(xc.const_data_ptr(), r, wc.const_data_ptr(), tag(dt), rows, H, (float)eps, hp,
                              y.mutable_data_ptr(), on.stream);
    return residual ? py::make_tuple(st, y, h) : py::make_tuple(st, y);
  }
  at::Tensor y = empty(x, x.sizes(), at::kFloat8_e4m3fn);
  c10::SmallVector<int64_t, 8> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = H / 128;
  at::Tensor s = empty(x, shape, e8m0 ? at::ScalarType::Float8_e8m0fnu : at::kFloat);
  const int st = p_rms_norm_quant(xc.const_data_ptr(), r, wc.const_data_ptr(), tag(dt), rows, H, (float)eps, pow2, hp,
                                  y.mutable_data_ptr(), s.mutable_data_ptr(), e8m0 ? BS_DT_E8M0 : BS_DT_F32, on.stream);
  return residual ? py::make_tuple(st, y, s, h) : py::make_tuple(st, y, s);
}

// The stride of dims 0..-3 taken as one, or -1 where they are not one.
int64_t token_stride(const at::Tensor& x) {
  int64_t stride = x.size(-1) * x.size(-2), want = -1;
  for (int64_t i = x.dim() - 3; i >= 0; --i) {
    if (x.size(i) == 1) continue;
    if (want < 0) stride = x.stride(i);
    else if (x.stride(i) != want) return -1;
    want = x.stride(i) * x.size(i);
  }
  return stride;
}

py::tuple rope(const at::Tensor& x, const at::Tensor& positions, const at::Tensor& freqs, bool half, int offset, bool inverse,
               double scale, bool inplace) {
  const On on(x, positions, freqs);
  const auto dt = x.scalar_type(), pt = positions.scalar_type();
  if (tag(dt) < 0) bad_type("rope: x is ", dt, ", expected bf16, f16 or fp32");
  if (pt != at::kLong && pt != at::kInt) bad_type("rope: positions are ", pt, ", expected int64 or int32");
  if (freqs.scalar_type() != at::kDouble || freqs.dim() != 1) bad_type("rope: freqs must be a float64 vector");
  if (x.dim() < 2 || positions.sizes() != x.sizes().slice(0, x.dim() - 2))
    bad_value("rope: positions ", positions.sizes(), " do not match x ", x.sizes());
  const int64_t H = x.size(-2), D = x.size(-1);
  if (H > INT_MAX || D > INT_MAX) bad_value("rope: x ", x.sizes());
  if (inplace && at::GradMode::is_enabled() && x.requires_grad())
    bad_value("rope: an in-place x requires a gradient, which would miss the turn");
  if (inplace && at::has_internal_overlap(x) == at::MemOverlap::Yes) bad_value("rope: an in-place x overlaps itself");
  at::Tensor xt = x;
  int64_t tok = H * D, head = D;
  if (!x.is_contiguous() || misaligned(x, 16)) {
    const int64_t e = 16 / x.element_size();
    tok = token_stride(x);
    head = x.stride(-2);
    if (tok < 0 || x.stride(-1) != 1 || head % e || tok % e || misaligned(x, 16)) {
      if (inplace) bad_value("rope: an in-place x needs contiguous 16-byte aligned dims and one stride over its tokens");
      xt = x.clone(at::MemoryFormat::Contiguous);
      tok = H * D;
      head = D;
    }
  }
  at::Tensor out = inplace ? x : empty(x, x.sizes(), dt);
  const auto pc = positions.expect_contiguous(), fc = freqs.expect_contiguous();
  const int st = p_rope(xt.const_data_ptr(), tag(dt), positions.numel(), (int)H, (int)D, tok, head, pc->const_data_ptr(),
                        pt == at::kLong, (const double*)fc->const_data_ptr(), (int)(2 * freqs.numel()), offset, half, inverse,
                        (float)scale, out.mutable_data_ptr(), inplace ? tok : H * D, inplace ? head : D, on.stream);
  if (inplace && st == BS_OK) changed(x);
  return py::make_tuple(st, out);
}

void check_cache(const char* name, const at::Tensor& cache, const at::Tensor& scale, int64_t D, int64_t Hkv) {
  if (cache.scalar_type() != at::kFloat8_e4m3fn || scale.scalar_type() != at::kFloat)
    bad_type(name, ": a cache is float8_e4m3fn with fp32 scales");
  if (cache.dim() != 4 || cache.size(1) != Hkv || cache.size(3) != D || scale.dim() != 2 || scale.size(0) != cache.size(0) ||
      scale.size(1) != Hkv)
    bad_value(name, ": cache ", cache.sizes(), " and scales ", scale.sizes(), " do not match [n_pages, ", Hkv, ", page, ", D, "]");
  if (!cache.is_contiguous() || !scale.is_contiguous()) bad_value(name, ": cache and scales must be contiguous");
}

at::Tensor index_arg(const char* name, const char* what, const at::Tensor& t, int64_t B, int64_t dims) {
  if (t.scalar_type() != at::kInt) bad_type(name, ": ", what, " is ", t.scalar_type(), ", expected int32");
  if (t.dim() != dims || t.size(0) != B) bad_value(name, ": ", what, " ", t.sizes(), ", expected ", dims, " dims of ", B, " sequences");
  return t.contiguous();
}

// x, or a contiguous copy where its strides do not keep vectors of `unit` elements whole.
at::Tensor strided(const at::Tensor& x, int64_t unit, uintptr_t align) {
  if (x.stride(3) == 1 && !(x.stride(0) % unit || x.stride(1) % unit || x.stride(2) % unit || misaligned(x, align))) return x;
  return x.clone(at::MemoryFormat::Contiguous);
}

int fits_int(const char* name, int64_t v) {
  if (v < 0 || v > INT_MAX) bad_value(name, ": size ", v);
  return (int)v;
}

int append(const at::Tensor& k, const Opt& v, const at::Tensor& k_cache, const Opt& v_cache, const at::Tensor& k_scale,
           const Opt& v_scale, const at::Tensor& block_table, const at::Tensor& start, const Opt& new_lens) {
  static const char* name = "cache_append";
  const On on(k, v, k_cache, v_cache, k_scale, v_scale, block_table, start, new_lens);
  if (k.dim() != 4) bad_value(name, ": k ", k.sizes(), ", expected [B, S, Hkv, D]");
  if (v.has_value() != v_cache.has_value() || v.has_value() != v_scale.has_value())
    bad_value(name, ": v, v_cache and v_scale go together");
  if (tag(k.scalar_type()) < 0 || (v && v->scalar_type() != k.scalar_type()))
    bad_type(name, ": k and v must have one type of bf16, f16 or fp32");
  const int64_t B = k.size(0), S = k.size(1), Hkv = k.size(2), D = k.size(3);
  check_cache(name, k_cache, k_scale, D, Hkv);
  if (v) {
    if (v->sizes() != k.sizes() || v_cache->sizes() != k_cache.sizes()) bad_value(name, ": v does not match k");
    check_cache(name, *v_cache, *v_scale, D, Hkv);
  }
  const at::Tensor bt = index_arg(name, "block_table", block_table, B, 2), st = index_arg(name, "start", start, B, 1);
  const at::Tensor nl = new_lens ? index_arg(name, "new_lens", *new_lens, B, 1) : at::Tensor();
  if (B == 0 || S == 0) return BS_OK;
  const int64_t e = 16 / k.element_size();
  const at::Tensor kc = strided(k, e, 16), vc = v ? strided(*v, e, 16) : at::Tensor();
  const int status = p_cache_append(kc.const_data_ptr(), v ? vc.const_data_ptr() : nullptr, tag(k.scalar_type()), B, S,
                                   fits_int(name, Hkv), fits_int(name, D), kc.strides().data(), v ? vc.strides().data() : nullptr,
                                   k_cache.mutable_data_ptr(), v ? v_cache->mutable_data_ptr() : nullptr,
                                   (float*)k_scale.mutable_data_ptr(), v ? (float*)v_scale->mutable_data_ptr() : nullptr,
                                   k_cache.size(0), fits_int(name, k_cache.size(2)), (const int*)bt.const_data_ptr(), bt.size(1),
                                   (const int*)st.const_data_ptr(), new_lens ? (const int*)nl.const_data_ptr() : nullptr, on.stream);
  if (status == BS_OK) {
    changed(k_cache);
    changed(k_scale);
    if (v) {
      changed(*v_cache);
      changed(*v_scale);
    }
  }
  return status;
}

py::tuple attn(const at::Tensor& q, const at::Tensor& k_cache, const Opt& v_cache, const at::Tensor& k_scale, const Opt& v_scale,
               const at::Tensor& block_table, const at::Tensor& seq_lens, double softmax_scale, const Opt& attn_sink,
               const Opt& new_lens) {
  static const char* name = "cache_attn";
  const On on(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, attn_sink, new_lens);
  if (q.dim() != 4) bad_value(name, ": q ", q.sizes(), ", expected [B, S, H, D]");
  const auto dt = q.scalar_type();
  if (dt != at::kBFloat16 && dt != at::kHalf) bad_type(name, ": q is ", dt, ", expected bf16 or f16");
  if (v_cache.has_value() != v_scale.has_value()) bad_value(name, ": v_cache and v_scale go together");
  if (k_cache.dim() != 4) bad_value(name, ": k_cache ", k_cache.sizes(), ", expected [n_pages, Hkv, page, D]");
  const int64_t B = q.size(0), S = q.size(1), H = q.size(2), D = q.size(3), Hkv = k_cache.size(1);
  check_cache(name, k_cache, k_scale, D, Hkv);
  if (v_cache) {
    check_cache(name, *v_cache, *v_scale, D, Hkv);
    if (v_cache->sizes() != k_cache.sizes()) bad_value(name, ": v_cache does not match k_cache");
  }
  if (Hkv == 0 || H % Hkv) bad_value(name, ": ", H, " query heads over ", Hkv, " kv heads");
  const at::Tensor bt = index_arg(name, "block_table", block_table, B, 2), sl = index_arg(name, "seq_lens", seq_lens, B, 1);
  const at::Tensor nl = new_lens ? index_arg(name, "new_lens", *new_lens, B, 1) : at::Tensor();
  at::Tensor sink;
  if (attn_sink) {
    if (attn_sink->dim() != 1 || attn_sink->size(0) != H) bad_value(name, ": attn_sink ", attn_sink->sizes(), ", expected [", H, "]");
    sink = attn_sink->to(at::kFloat).contiguous();
  }
  at::Tensor out = empty(q, q.sizes(), dt);
  if (out.numel() == 0) return py::make_tuple((int)BS_OK, out);
  const at::Tensor qc = strided(q, 4, 8);
  const int h = fits_int(name, H), hkv = fits_int(name, Hkv), d = fits_int(name, D);
  const size_t n = p_cache_attn_ws(B, S, h, hkv, d, tag(dt));
  const at::Tensor ws = empty(q, {(int64_t)(n ? n : 256)}, at::kByte);
  const int st = p_cache_attn(qc.const_data_ptr(), tag(dt), B, S, h, hkv, d, qc.strides().data(), k_cache.const_data_ptr(),
                              ptr(v_cache), (const float*)k_scale.const_data_ptr(), (const float*)ptr(v_scale),
                              k_cache.size(0), fits_int(name, k_cache.size(2)), (const int*)bt.const_data_ptr(), bt.size(1),
                              (const int*)sl.const_data_ptr(), new_lens ? (const int*)nl.const_data_ptr() : nullptr,
                              attn_sink ? (const float*)sink.const_data_ptr() : nullptr, (float)softmax_scale,
                              out.mutable_data_ptr(), ws.mutable_data_ptr(), ws.numel(), on.stream);
  return py::make_tuple(st, out);
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.def("bind", &bind);
  m.def("rms", &rms);
  m.def("rope", &rope);
  m.def("append", &append);
  m.def("attn", &attn);
}
