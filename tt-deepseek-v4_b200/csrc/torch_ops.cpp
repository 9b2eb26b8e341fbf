// The low-bit operators over torch tensors: argument checks, allocation of
// what the caller does not pass, the current stream, then the C ABI
// (include/dsv4attn.h).  Compiled, because a decode step calls them with
// kernels of 2-10 us: through ctypes a call took the host 12-19 us, here 2.8
// (cache write) to 7.6 (projection of 64 tokens, two launches and two
// allocations); a launch is ~2 of it.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "dsv4attn.h"

namespace py = pybind11;
using at::Tensor;
using Opt = std::optional<Tensor>;

namespace {

template <typename... A>
[[noreturn]] void bad(const A&... a) {
  throw py::value_error(c10::str(a...));
}

// Runs a call of the C ABI without the interpreter's lock (a launch waits
// while the device's queue is full) and maps its status as _lib.check does.
template <typename F>
void call(const char* what, F&& f) {
  int rc;
  {
    py::gil_scoped_release no_gil;
    rc = f();
  }
  if (rc == DSA_OK) return;
  const char* m = dsa_last_error();
  const std::string msg = std::string(what) + ": " + (m && *m ? m : ("status " + std::to_string(rc)).c_str());
  if (rc == DSA_ERR_ARG || rc == DSA_ERR_WORKSPACE || rc == DSA_ERR_UNSUPPORTED) throw py::value_error(msg);
  PyErr_SetString(rc == DSA_ERR_TIMEOUT ? PyExc_TimeoutError : PyExc_RuntimeError, msg.c_str());
  throw py::error_already_set();
}

std::string dtype_name(at::ScalarType t) {
  return py::cast<std::string>(py::str(py::reinterpret_borrow<py::object>(
      reinterpret_cast<PyObject*>(torch::getTHPDtype(t)))));
}

void need(const Tensor& t, const char* name) {
  if (!t.is_cuda()) bad(name, " must be a CUDA tensor (no CPU fallback)");
}
void need(const Tensor& t, const char* name, at::ScalarType dtype) {
  need(t, name);
  if (t.scalar_type() != dtype) bad(name, " must be ", dtype_name(dtype), ", got ", dtype_name(t.scalar_type()));
}
void contig(const Tensor& t, const char* name) {
  if (!t.is_contiguous()) bad(name, " must be contiguous");
}

int x_type(const Tensor& x) {
  switch (x.scalar_type()) {
    case at::kBFloat16: return DSA_BF16;
    case at::kHalf: return DSA_FP16;
    case at::kFloat: return DSA_FP32;
    default: bad("x must be bfloat16, float16 or float32, got ", dtype_name(x.scalar_type()));
  }
}

// row stride of t [..., K] read as a matrix of rows with unit stride
int64_t row_stride(const Tensor& t, const char* name) {
  const int64_t K = t.size(-1), d = t.dim();
  if (t.is_contiguous()) return K;
  if (t.stride(-1) != 1 && K > 1) bad(name, " must have a unit stride in the last dim");
  // the leading dims collapse into one: the innermost of size > 1 sets the
  // stride, each further one must continue it
  int64_t ld = -1, expect = 0;
  for (int64_t i = d - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (ld < 0)
      ld = t.stride(i);
    else if (t.stride(i) != expect)
      bad(name, " ", t.sizes(), " with strides ", t.strides(), " is not a matrix of rows");
    expect = t.stride(i) * t.size(i);
  }
  return ld < 0 ? K : ld;
}

// The current stream of t's device.  Launches go to the current device: t and
// the other tensors must be on it.
dsa_stream_t launch_stream(const Tensor& t, std::initializer_list<const Tensor*> others) {
  const auto dev = t.get_device();
  for (const Tensor* o : others)
    if (o && o->get_device() != dev) bad("tensors on ", t.device(), " and ", o->device());
  if (dev != c10::cuda::current_device())
    bad("tensor on ", t.device(), ", current device is cuda:", int(c10::cuda::current_device()));
  return reinterpret_cast<dsa_stream_t>(c10::cuda::getCurrentCUDAStream(dev).stream());
}

const Tensor* ptr(const Opt& t) { return t ? &*t : nullptr; }
template <typename T = void>
T* data(const Opt& t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}
int32_t* status_of(const Opt& t) {
  if (t) need(*t, "status", at::kInt);
  return data<int32_t>(t);
}

// Past the dispatcher, 0.3-0.4 us a tensor less (a quantisation's three: 6.4 ->
// 5.6 us a call).  What it leaves out besides, the deterministic mode's fill,
// is not needed: every element is written.
Tensor empty_like_type(at::IntArrayRef shape, const Tensor& t, at::ScalarType dtype) {
  return at::detail::empty_cuda(shape, dtype, t.device(), std::nullopt);
}

// scratch: from the caller's Workspace, or of the current stream
Tensor scratch(const py::object& ws, size_t bytes, const Tensor& like) {
  if (!ws.is_none()) {
    Tensor buf = py::cast<Tensor>(ws.attr("get")(bytes));
    if (buf.device() != like.device()) bad("workspace on ", buf.device(), ", tensors on ", like.device());
    return buf;
  }
  return empty_like_type({int64_t(bytes)}, like, at::kByte);
}

py::tuple mxfp4_quant(const Tensor& x, const py::object& out_arg, Opt codes, Opt scales) {
  need(x, "x");
  const int type = x_type(x);
  const int64_t K = x.dim() ? x.size(-1) : 0;
  if (K == 0 || K % 32) bad("last dim ", K, " must be a positive multiple of 32");
  const int64_t ld = row_stride(x, "x");
  Opt out;
  const bool make = out_arg.ptr() == Py_True;
  if (!make && !out_arg.is_none()) {
    if (!THPVariable_Check(out_arg.ptr())) throw py::type_error("out must be a tensor, True or None");
    out = py::cast<Tensor>(out_arg);
  }
  const auto stream = launch_stream(x, {ptr(out), ptr(codes), ptr(scales)});
  int64_t ld_out = K;
  if (make) {
    out = empty_like_type(x.sizes(), x, x.scalar_type());
  } else if (out) {
    need(*out, "out", x.scalar_type());
    if (out->sizes() != x.sizes()) bad("out must have x's shape");
    ld_out = row_stride(*out, "out");
  }
  std::vector<int64_t> shape = x.sizes().vec();
  auto field = [&](Opt& t, const char* name, int64_t w) {
    shape.back() = w;
    if (!t) {
      t = empty_like_type(shape, x, at::kByte);
      return;
    }
    need(*t, name, at::kByte);
    contig(*t, name);
    if (t->sizes() != at::IntArrayRef(shape)) bad(name, " must be ", at::IntArrayRef(shape), ", got ", t->sizes());
  };
  field(codes, "codes", K / 2);
  field(scales, "scales", K / 32);
  const int64_t M = x.numel() / K;
  if (M)
    call("mxfp4_quant", [&] {
      return dsa_mxfp4_quant(x.data_ptr(), type, ld, data(out), ld_out, data<uint8_t>(codes), data<uint8_t>(scales),
                             M, K, stream);
    });
  return py::make_tuple(out ? py::cast(*out) : py::none(), *scales, *codes);
}

Tensor linear_mxfp4(const Tensor& x, const Tensor& packed, int64_t N, int64_t K, const Opt& out_arg, bool out_f32,
                    const py::object& ws, const Opt& status) {
  // the product reads every tile that N and K name
  const size_t tiles = N > 0 && N <= INT32_MAX && K > 0 && K <= INT32_MAX ? dsa_linear_mxfp4_packed_bytes(int(N), int(K)) : 0;
  if (tiles == 0 || packed.scalar_type() != at::kByte || !packed.is_contiguous() || size_t(packed.numel()) < tiles)
    bad("w's packed tensor must be the tiles of a [", N, ", ", K, "] weight (contiguous uint8, ", tiles,
        " bytes), got ", dtype_name(packed.scalar_type()), " ", packed.sizes());
  need(x, "x");
  const int type = x_type(x);
  if (x.dim() != 2 || x.size(1) != K || x.stride(1) != 1)
    bad("x must be [B, ", K, "] with contiguous rows, got ", x.sizes());
  const int64_t B = x.size(0);
  const auto dtype = out_f32 ? at::kFloat : at::kBFloat16;
  const auto stream = launch_stream(x, {&packed, ptr(out_arg), ptr(status)});
  int32_t* st = status_of(status);
  if (B > INT32_MAX) bad("x has too many rows");
  Tensor out;
  if (!out_arg) {
    out = empty_like_type({B, N}, x, dtype);
  } else {
    out = *out_arg;
    need(out, "out", dtype);
    if (out.dim() != 2 || out.size(0) != B || out.size(1) < N || out.stride(1) != 1)
      bad("out must be [", B, ", >=", N, "] with contiguous rows, got ", out.sizes());
  }
  if (B == 0) return out;
  const size_t bytes = dsa_linear_mxfp4_workspace_size(int(B), int(N), int(K));
  Tensor buf;
  if (bytes) buf = scratch(ws, bytes, x);
  call("linear_mxfp4", [&] {
    return dsa_linear_mxfp4(x.data_ptr(), type, x.stride(0), packed.data_ptr(), out.data_ptr(), out.stride(0), int(B),
                            int(N), int(K), out_f32, bytes ? buf.data_ptr() : nullptr, bytes, st, stream);
  });
  return out;
}

int64_t row_bytes(int64_t D, int64_t rope_dim) {
  const int64_t n = D > 0 && D <= 8192 && rope_dim >= 0 && rope_dim < D
                        ? int64_t(dsa_kv_quant_row_bytes(int(D), int(rope_dim)))
                        : 0;
  if (n == 0)
    bad("D=", D, ", rope_dim=", rope_dim,
        ": D - rope_dim must be a positive multiple of 64, rope_dim a multiple of 8, D <= 8192");
  return n;
}

py::tuple kv_quant_views(const Tensor& cache, int64_t D, int64_t rope_dim) {
  const int64_t rb = row_bytes(D, rope_dim), a = D - rope_dim, b = a + 2 * rope_dim;
  if (cache.scalar_type() != at::kByte || cache.dim() == 0 || cache.size(-1) != rb)
    bad("cache must be uint8 with records of ", rb, " bytes");
  return py::make_tuple(cache.narrow(-1, 0, a).view(at::kFloat8_e4m3fn), cache.narrow(-1, a, b - a).view(at::kBFloat16),
                        cache.narrow(-1, b, a / 16).view(at::kFloat));
}

void quant_cache(const Tensor& cache, int64_t B, int64_t D, int64_t rope_dim) {
  need(cache, "cache", at::kByte);
  const int64_t rb = row_bytes(D, rope_dim);
  if (cache.dim() != 3 || cache.size(0) < B || cache.size(1) < 1 || cache.size(2) != rb || cache.stride(2) != 1 ||
      (cache.size(1) > 1 && cache.stride(1) != rb))
    bad("cache must be [>=", B, ", rows, ", rb, "] with contiguous rows (D=", D, ", rope_dim=", rope_dim, "), got ",
        cache.sizes());
}

// bytes between sequences; of one sequence nothing steps by it
int64_t cache_stride(const Tensor& cache, int64_t B) {
  return B > 1 ? cache.stride(0) : cache.size(1) * cache.size(2);
}

void per_sequence(const Tensor& t, const char* name, int64_t B) {
  need(t, name, at::kInt);
  contig(t, name);
  if (t.numel() != B) bad(name, " has ", t.numel(), " entries, expected ", B);
}

void kv_quant_write(const Tensor& kv_arg, const Tensor& cache, const Tensor& pos, int64_t win, int64_t offset,
                    int64_t rope_dim, const Opt& n_valid) {
  need(kv_arg, "kv", at::kBFloat16);
  const int64_t d = kv_arg.dim();
  if ((d != 2 && d != 3) || kv_arg.stride(-1) != 1)
    bad("kv must be [B, S, D] or [B, D] with a unit stride in the last dim");
  const int64_t B = kv_arg.size(0), S = d == 3 ? kv_arg.size(1) : 1, D = kv_arg.size(-1);
  const int64_t ld_b = B > 1 ? kv_arg.stride(0) : 0, ld_s = S > 1 ? kv_arg.stride(1) : 0;
  quant_cache(cache, B, D, rope_dim);
  per_sequence(pos, "pos", B);
  if (n_valid) per_sequence(*n_valid, "n_valid", B);
  const auto stream = launch_stream(kv_arg, {&cache, &pos, ptr(n_valid)});
  if (B > INT32_MAX || S > INT32_MAX || win != int32_t(win)) bad("kv_quant_write: B, S or win is too large");
  if (B && S)
    call("kv_quant_write", [&] {
      return dsa_kv_quant_write(kv_arg.data_ptr(), ld_b, ld_s, cache.data_ptr(), cache_stride(cache, B), cache.size(1),
                                static_cast<const int32_t*>(pos.data_ptr()), data<const int32_t>(n_valid), int(B),
                                int(S), int(D), int(rope_dim), int(win), offset, stream);
    });
}

Tensor kv_quant_read(const Tensor& cache, const Opt& idx, int64_t D, int64_t rope_dim, at::ScalarType dtype,
                     const Opt& out_arg, const Opt& status) {
  quant_cache(cache, 0, D, rope_dim);
  const int64_t B = cache.size(0);
  if (dtype != at::kBFloat16 && dtype != at::kFloat)
    bad("dtype must be bfloat16 or float32, got ", dtype_name(dtype));
  int64_t K = cache.size(1), ld = 0;
  if (idx) {
    need(*idx, "idx", at::kInt);
    if (idx->dim() != 2 || idx->size(0) != B || (idx->stride(1) != 1 && idx->size(1) > 1))
      bad("idx must be [", B, ", K] with a unit stride in the last dim");
    K = idx->size(1);
    ld = B > 1 ? idx->stride(0) : K;
  }
  const auto stream = launch_stream(cache, {ptr(idx), ptr(out_arg), ptr(status)});
  int32_t* st = status_of(status);
  Tensor out;
  if (!out_arg) {
    out = empty_like_type({B, K, D}, cache, dtype);
  } else {
    out = *out_arg;
    need(out, "out", dtype);
    contig(out, "out");
    const int64_t want[3] = {B, K, D};
    if (out.sizes() != at::IntArrayRef(want, 3)) bad("out must be ", at::IntArrayRef(want, 3), ", got ", out.sizes());
  }
  if (B > INT32_MAX) bad("kv_quant_read: B is too large");
  if (B && K)
    call("kv_quant_read", [&] {
      return dsa_kv_quant_read(cache.data_ptr(), cache_stride(cache, B), cache.size(1), data<const int32_t>(idx), ld,
                               out.data_ptr(), dtype == at::kFloat, int(B), K, int(D), int(rope_dim), st, stream);
    });
  return out;
}

Tensor sparse_attn_quant(const Tensor& q, const Tensor& cache, const Tensor& idx, const Tensor& sink, double scale,
                         const Opt& out_arg, const Opt& lse, const py::object& ws, const Opt& status) {
  need(q, "q", at::kBFloat16);
  contig(q, "q");
  need(idx, "idx", at::kInt);
  need(sink, "sink", at::kFloat);
  contig(sink, "sink");
  const int64_t d = q.dim();
  if (d != 3 && d != 4) bad("q must be [B, S, H, D] or [B, H, D]");
  const int64_t B = q.size(0), S = d == 4 ? q.size(1) : 1, H = q.size(-2), D = q.size(-1);
  if (H != 64 || D != 512 || sink.numel() != H)
    bad("sparse_attn_quant: built for 64 heads of 512 dims and as many sinks (got ", H, " of ", D, ", ", sink.numel(),
        " sinks)");
  quant_cache(cache, B, D, 64);
  const int64_t di = idx.dim();
  const bool rows3 = di == 3 && idx.size(0) == B && idx.size(1) == S;
  const bool rows2 = di == 2 && S == 1 && idx.size(0) == B;
  if (!rows3 && !rows2) bad("idx must be [B, S, K] for q ", q.sizes(), ", got ", idx.sizes());
  const int64_t K = idx.size(-1);
  const int64_t ld_idx = K ? row_stride(idx, "idx") : 0;
  const auto stream = launch_stream(q, {&cache, &idx, &sink, ptr(out_arg), ptr(lse), ptr(status)});
  int32_t* st = status_of(status);
  Tensor out;
  if (!out_arg) {
    out = empty_like_type(q.sizes(), q, at::kBFloat16);
  } else {
    out = *out_arg;
    need(out, "out", at::kBFloat16);
    contig(out, "out");
    if (out.sizes() != q.sizes()) bad("out must have q's shape");
  }
  if (lse) {
    need(*lse, "lse", at::kFloat);
    contig(*lse, "lse");
    if (lse->numel() != B * S * H) bad("lse has ", lse->numel(), " elements, expected ", B * S * H);
  }
  if (B == 0 || S == 0) return out;
  if (B * S > 65535 || K > INT32_MAX) bad("sparse_attn_quant: B*S = ", B * S, " query rows is too many (65535 a call)");
  const size_t bytes = dsa_sparse_attn_workspace_size(int(B), int(S), int(H), int(D), int(K));
  Tensor buf;
  if (bytes) buf = scratch(ws, bytes, q);
  call("sparse_attn_quant", [&] {
    return dsa_sparse_attn_quant(q.data_ptr(), cache.data_ptr(), cache_stride(cache, B), cache.size(1),
                                 static_cast<const int32_t*>(K ? idx.data_ptr() : sink.data_ptr()), ld_idx,
                                 static_cast<const float*>(sink.data_ptr()), out.data_ptr(), data<float>(lse), int(B),
                                 int(S), int(H), int(D), int(K), float(scale), bytes ? buf.data_ptr() : nullptr, bytes,
                                 st, stream);
  });
  return out;
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  m.def("mxfp4_quant", &mxfp4_quant);
  m.def("linear_mxfp4", &linear_mxfp4);
  m.def("kv_quant_row_bytes", &row_bytes);
  m.def("kv_quant_views", &kv_quant_views);
  m.def("kv_quant_write", &kv_quant_write);
  m.def("kv_quant_read", &kv_quant_read);
  m.def("sparse_attn_quant", &sparse_attn_quant);
}
