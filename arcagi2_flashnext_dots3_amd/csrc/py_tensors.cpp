// The norm, quantization, projection, rotary and latent-row calls on tensors: checks of shapes, types, strides and devices,
// then the entry point (include/spmla.h) on the current stream. _tensors.load(path, raw_stream, get_device) opens the
// library and returns {name: callable}; a callable raises ValueError for what the call does not take, before it launches
// anything, and returns the entry point's value, or AWAY when the tensors are on another GPU than the current one. These
// calls are a few us on the GPU: the same checks in Python took 4 us of 7, here 0.4.
#include <ATen/ATen.h>
#include <Python.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdexcept>
#include <string>

#include "spmla.h"
#include "spmla_rules.h"

namespace {

constexpr long AWAY = -1000;

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
[[noreturn]] void refuse(const std::string& what) { throw Refused(what); }
struct Raised {};      // a Python error is set

decltype(&::spmla_rms_norm) f_rms_norm = nullptr;
decltype(&::spmla_quant_fp8) f_quant_fp8 = nullptr;
decltype(&::spmla_linear_fp8) f_linear_fp8 = nullptr;
decltype(&::spmla_rope) f_rope = nullptr;
decltype(&::spmla_latent_write) f_latent_write = nullptr;
PyObject *raw_stream = nullptr, *get_device = nullptr;

// ---- arguments
const at::Tensor* tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + ": a tensor expected, got " + Py_TYPE(o)->tp_name);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != at::kStrided) refuse(std::string(name) + ": a dense tensor expected");
  return &t;
}
const at::Tensor* maybe(PyObject* o, const char* name) { return o == Py_None ? nullptr : tensor(o, name); }
double number(PyObject* o) {
  const double d = PyFloat_AsDouble(o);
  if (d == -1.0 && PyErr_Occurred()) throw Raised{};
  return d;
}
long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised{};
  return v != 0;
}
int as_int(int64_t v, const char* name) {
  if (v > 0x7fffffff || v < -0x7fffffff - 1) refuse(std::string(name) + " of " + std::to_string(v) + ": 32 bits");
  return (int)v;
}

// ---- checks
enum : unsigned { F32 = 1, F16 = 2, BF16 = 4, E4M3 = 8, U8 = 16, I32 = 32, I64 = 64, F64 = 128, OTHER = 0 };
unsigned type_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return F32;
    case at::kHalf: return F16;
    case at::kBFloat16: return BF16;
    case at::kFloat8_e4m3fn: return E4M3;
    case at::kByte: return U8;
    case at::kInt: return I32;
    case at::kLong: return I64;
    case at::kDouble: return F64;
    default: return OTHER;
  }
}
int dtype_code(unsigned type) { return type == F32 ? 0 : type == F16 ? 1 : 2; }    // the C-ABI's dtype argument
int gpu_of(const at::Tensor& t) { return t.is_cuda() ? (int)t.get_device() : -1; }
void same_gpu(const at::Tensor& t, int dev, const char* name) {
  if (dev < 0 || gpu_of(t) != dev) refuse(std::string(name) + ": tensors on one GPU");
}
std::string shown(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t n : t.sizes()) s += std::to_string(n) + ", ";
  return s + ") " + c10::toString(t.scalar_type());
}
void* address(const at::Tensor* t) { return t ? const_cast<void*>(t->const_data_ptr()) : nullptr; }

// row stride of t [T, D] with contiguous rows (a single row's is D, whatever its tensor says); written: rows that do not overlap
int64_t rows(const at::Tensor& t, int64_t T, int64_t D, unsigned types, const char* what, bool written = false) {
  if (t.dim() != 2 || t.size(0) != T || t.size(1) != D || !(type_of(t) & types))
    refuse(std::string(what) + " expected, (" + std::to_string(T) + ", " + std::to_string(D) + "): got " + shown(t));
  if (D > 1 && t.stride(1) != 1) refuse(std::string(what) + ": contiguous rows");
  if (written && T > 1 && t.stride(0) < D) refuse(std::string(what) + ": rows that do not overlap");
  return T > 1 ? t.stride(0) : D;
}
void line(const at::Tensor& t, int64_t least, int64_t most, unsigned types, const char* what) {
  if (t.dim() != 1 || t.size(0) < least || t.size(0) > most || !(type_of(t) & types) || !t.is_contiguous())
    refuse(std::string(what) + " expected: got " + shown(t));
}
constexpr int64_t ANY = INT64_MAX;
void on_bytes(const at::Tensor& t, int64_t stride_bytes, int bytes, const char* what) {   // address and rows
  if (((uintptr_t)t.const_data_ptr() | (uint64_t)stride_bytes) & (bytes - 1))
    refuse(std::string(what) + ": rows on " + std::to_string(bytes) + " bytes");
}
void at_most(int64_t v, int64_t most, const char* name) {
  if (v > most) refuse(std::string(name) + " of " + std::to_string(v) + ": at most " + std::to_string(most));
}
constexpr int64_t MAX_TOKENS = 1 << 23;
float epsilon(double eps) {
  if (!((float)eps >= 0.f)) refuse("eps >= 0: got " + std::to_string(eps));
  return (float)eps;
}

// the current stream of dev as an address, or AWAY's flag
bool stream_of(int dev, void*& s) {
  PyObject* cur = PyObject_CallNoArgs(get_device);
  if (!cur) throw Raised{};
  const long at = PyLong_AsLong(cur);
  Py_DECREF(cur);
  if (at != dev) return false;
  PyObject* arg = PyLong_FromLong(dev);
  PyObject* v = arg ? PyObject_CallOneArg(raw_stream, arg) : nullptr;
  Py_XDECREF(arg);
  if (!v) throw Raised{};
  s = PyLong_AsVoidPtr(v);
  Py_DECREF(v);
  if (PyErr_Occurred()) throw Raised{};
  return true;
}

template <class F>
long launch(int dev, F f) {
  void* s = nullptr;
  if (!stream_of(dev, s)) return AWAY;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f(s);
  Py_END_ALLOW_THREADS
  return rc;
}

struct Norm {                                            // shape and type of a norm's or quantization's input
  const at::Tensor* x;
  int64_t T, D, st;
  unsigned type;
  int dev;
};
Norm norm_input(PyObject* o) {
  const at::Tensor* x = tensor(o, "x");
  const unsigned type = type_of(*x);
  if (x->dim() != 2 || !(type & (F32 | F16 | BF16)) || x->size(1) == 0) refuse("x [T, D] fp32 / fp16 / bf16, D > 0: got " + shown(*x));
  Norm n{x, x->size(0), x->size(1), 0, type, gpu_of(*x)};
  n.st = rows(*x, n.T, n.D, type, "x [T, D]");
  at_most(n.T, MAX_TOKENS, "T");
  return n;
}
constexpr const char* CODES = "codes [T, D] e4m3 / uint8";
constexpr const char* SCALES = "scales [T, ceil(D / 128)] fp32";

// rms_norm(x, weight, eps, residual, residual_out, out, codes, scales, ue8m0)
long rms_norm(PyObject* const* a) {
  const Norm n = norm_input(a[0]);
  const at::Tensor *w = maybe(a[1], "weight"), *r = maybe(a[3], "residual"), *ro = maybe(a[4], "residual_out");
  const at::Tensor *out = maybe(a[5], "out"), *codes = maybe(a[6], "codes"), *scales = maybe(a[7], "scales");
  const float eps = epsilon(number(a[2]));
  const bool ue8m0 = truth(a[8]);
  at_most(n.D, 65536, "D");
  int64_t rs = 0, ros = 0, os = 0, cs = 0, ss = 0;
  if (r) {
    rs = rows(*r, n.T, n.D, n.type, "residual [T, D] of x's type");
    if (!ro) ro = r;
    ros = rows(*ro, n.T, n.D, n.type, "residual_out [T, D] of x's type", true);
  } else if (ro) {
    refuse("residual_out without a residual");
  }
  if (w) line(*w, n.D, n.D, n.type | F32, "weight [D] of x's type or fp32");
  if (out) os = rows(*out, n.T, n.D, n.type, "out [T, D] of x's type", true);
  if (codes) {
    cs = rows(*codes, n.T, n.D, E4M3 | U8, CODES, true);
    if (!scales) refuse("codes without scales");
    ss = rows(*scales, n.T, (n.D + 127) / 128, F32, SCALES, true);
  }
  for (const at::Tensor* t : {n.x, w, r, ro, out, codes, scales})
    if (t) same_gpu(*t, n.dev, "rms_norm");
  const int T = as_int(n.T, "T"), D = as_int(n.D, "D"), wf = w && type_of(*w) == F32;
  return launch(n.dev, [&](void* s) {
    return f_rms_norm(address(n.x), n.st, address(r), rs, address(ro), ros, address(w), wf, eps, T, D, dtype_code(n.type),
                      address(out), os, (unsigned char*)address(codes), cs, (float*)address(scales), ss, ue8m0, s);
  });
}

// quant_fp8(x, codes, scales, ue8m0)
long quant_fp8(PyObject* const* a) {
  const Norm n = norm_input(a[0]);
  const at::Tensor *codes = tensor(a[1], "codes"), *scales = tensor(a[2], "scales");
  const bool ue8m0 = truth(a[3]);
  at_most(n.D, 65535 * 2048, "D");
  const int64_t cs = rows(*codes, n.T, n.D, E4M3 | U8, CODES, true);
  const int64_t ss = rows(*scales, n.T, (n.D + 127) / 128, F32, SCALES, true);
  for (const at::Tensor* t : {n.x, codes, scales}) same_gpu(*t, n.dev, "quant_fp8");
  const int T = as_int(n.T, "T"), D = as_int(n.D, "D");
  return launch(n.dev, [&](void* s) {
    return f_quant_fp8(address(n.x), n.st, T, D, dtype_code(n.type), (unsigned char*)address(codes), cs, (float*)address(scales),
                       ss, ue8m0, s);
  });
}

constexpr const char *WEIGHT = "w [N, K] e4m3", *WEIGHT_SCALES = "w_scales [ceil(N / 128), ceil(K / 128)] fp32";
constexpr const char* PRODUCT = "out [T, N] bf16 / fp16";
constexpr int64_t MAX_K = 1 << 22;

struct Weight {                                          // a projection's weight and scales, for T rows of K values
  int64_t N, w_st, ws_st;
};
Weight weight(const at::Tensor& w, const at::Tensor& ws, int64_t T, int64_t K) {
  const int64_t N = w.size(0), kb = (K + 127) / 128;
  if (K == 0 || K % 16) refuse("K a positive multiple of 16: got " + std::to_string(K));
  const Weight f{N, rows(w, N, K, E4M3 | U8, WEIGHT, true), rows(ws, (N + 127) / 128, kb, F32, WEIGHT_SCALES, true)};
  if (T == 0 || N == 0) return f;
  on_bytes(w, f.w_st, 16, WEIGHT);
  at_most(T, MAX_TOKENS, "T");
  at_most(N, MAX_TOKENS, "N");
  at_most(K, MAX_K, "K");
  at_most(f.w_st, MAX_K, "stride of w");
  // tiles of 16 x 16 are the most workgroups: where these are many, the rule says
  if ((T / 16 + 1) * (N / 16 + 1) >= 1 << 22 && spmla::rules::linear_kernel((int)T, (int)N, (int)K) < 0)
    refuse("T, N of " + std::to_string(T) + ", " + std::to_string(N) + ": more tiles than one launch takes");
  return f;
}

// linear_fp8(a, a_scales, w, w_scales, out)
long linear_fp8(PyObject* const* v) {
  const at::Tensor *a = tensor(v[0], "a"), *as = tensor(v[1], "a_scales"), *w = tensor(v[2], "w");
  const at::Tensor *ws = tensor(v[3], "w_scales"), *out = tensor(v[4], "out");
  if (a->dim() != 2 || w->dim() != 2 || a->size(1) != w->size(1)) refuse("a [T, K], w [N, K]: got " + shown(*a) + ", " + shown(*w));
  const int64_t T = a->size(0), K = a->size(1), kb = (K + 127) / 128;
  const Weight f = weight(*w, *ws, T, K);
  const int64_t N = f.N;
  const int64_t a_st = rows(*a, T, K, E4M3 | U8, "a [T, K] e4m3", true);
  const int64_t as_st = rows(*as, T, kb, F32, "a_scales [T, ceil(K / 128)] fp32", true);
  if (T > 0 && N > 0) {
    on_bytes(*a, a_st, 16, "a [T, K] e4m3");
    at_most(a_st, MAX_K, "stride of a");
    at_most(as_st, 1 << 20, "stride of a_scales");
  }
  const int64_t o_st = rows(*out, T, N, BF16 | F16, PRODUCT, true);
  const int dev = gpu_of(*a);
  for (const at::Tensor* t : {a, as, w, ws, out}) same_gpu(*t, dev, "linear_fp8");
  const int Ti = as_int(T, "T"), Ni = as_int(N, "N"), Ki = as_int(K, "K");
  return launch(dev, [&](void* s) {
    return f_linear_fp8(address(a), a_st, (const float*)address(as), as_st, address(w), f.w_st, (const float*)address(ws), f.ws_st,
                        Ti, Ni, Ki, dtype_code(type_of(*out)), address(out), o_st, s);
  });
}

// linear_quant(x, w, w_scales, out, work, ue8m0): quant_fp8 into work (T K bytes of codes, then the scales), then linear_fp8
long linear_quant(PyObject* const* v) {
  const Norm n = norm_input(v[0]);
  const at::Tensor *w = tensor(v[1], "w"), *ws = tensor(v[2], "w_scales"), *out = tensor(v[3], "out"), *work = tensor(v[4], "work");
  const bool ue8m0 = truth(v[5]);
  if (w->dim() != 2 || n.D != w->size(1)) refuse("x [T, K], w [N, K]: got " + shown(*n.x) + ", " + shown(*w));
  const Weight f = weight(*w, *ws, n.T, n.D);
  const int64_t N = f.N, kb = (n.D + 127) / 128;
  const int64_t o_st = rows(*out, n.T, N, BF16 | F16, PRODUCT, true);
  line(*work, n.T * (n.D + 4 * kb), ANY, U8, "work [T (K + 4 ceil(K / 128))] uint8");
  for (const at::Tensor* t : {n.x, w, ws, out, work}) same_gpu(*t, n.dev, "linear_fp8");
  const int T = as_int(n.T, "T"), Ni = as_int(N, "N"), K = as_int(n.D, "K");
  unsigned char* codes = (unsigned char*)address(work);
  float* scales = (float*)(codes + n.T * n.D);
  return launch(n.dev, [&](void* s) {
    const int rc = f_quant_fp8(address(n.x), n.st, T, K, dtype_code(n.type), codes, n.D, scales, kb, ue8m0, s);
    return rc ? rc : f_linear_fp8(codes, n.D, scales, kb, address(w), f.w_st, (const float*)address(ws), f.ws_st, T, Ni, K,
                                  dtype_code(type_of(*out)), address(out), o_st, s);
  });
}

// rope(x, positions, freqs, out, start, interleaved, factor, inverse)
long rope(PyObject* const* a) {
  const at::Tensor *x = tensor(a[0], "x"), *pos = tensor(a[1], "positions"), *freqs = tensor(a[2], "freqs"), *out = tensor(a[3], "out");
  const long long start = integer(a[4]);
  const bool inter = truth(a[5]), inverse = truth(a[7]);
  const double factor = number(a[6]);
  const int64_t d = x->dim();
  const unsigned type = type_of(*x);
  if ((d != 2 && d != 3) || !(type & (F32 | F16 | BF16))) refuse("x [T, H, W] or [T, W] fp32 / fp16 / bf16: got " + shown(*x));
  if (out->sizes() != x->sizes() || type_of(*out) != type) refuse("out of x's shape and type: got " + shown(*out));
  const int64_t T = x->size(0), H = d == 3 ? x->size(1) : 1, W = x->size(d - 1);
  auto stride = [](const at::Tensor& t, int64_t i) -> int64_t { return t.size(i) > 1 ? t.stride(i) : 0; };   // a single one's says nothing
  const int64_t x_st = stride(*x, 0), o_st = stride(*out, 0), x_sh = d == 3 ? stride(*x, 1) : 0, o_sh = d == 3 ? stride(*out, 1) : 0;
  if (W > 1 && (x->stride(d - 1) != 1 || out->stride(d - 1) != 1)) refuse("contiguous head columns");
  line(*pos, T, ANY, I32 | I64, "positions [T] int32 / int64");
  line(*freqs, 0, ANY, F64, "freqs [pairs] float64");
  const int64_t n = freqs->size(0);
  if (start < 0 || n > W / 2 || start > W - 2 * n) refuse("start + 2 len(freqs) columns inside the head");
  // heads of a token or tokens of a head lie behind one another: no element is written twice
  if (T > 0 && H > 0 && ((T > 1 && o_st < W) || (H > 1 && o_sh < W) ||
                         (T > 1 && H > 1 && o_st < (H - 1) * o_sh + W && o_sh < (T - 1) * o_st + W)))
    refuse("out: heads that do not overlap");
  if (T > 0 && H > 0 && W > 0 && address(out) == address(x) && (x_st != o_st || x_sh != o_sh)) refuse("out: x's strides where it is x itself");
  at_most(T, MAX_TOKENS, "T");
  at_most(H, 1 << 30, "H");
  at_most(W, 1 << 30, "W");
  const int dev = gpu_of(*x);
  for (const at::Tensor* t : {x, pos, freqs, out}) same_gpu(*t, dev, "rope");
  const int Ti = as_int(T, "T"), Hi = as_int(H, "H"), Wi = as_int(W, "W");
  return launch(dev, [&](void* s) {
    return f_rope(address(x), x_st, x_sh, address(pos), type_of(*pos) == I32, (const double*)address(freqs), Ti, Hi, Wi, (int)start,
                  (int)n, inter, (float)factor, inverse, dtype_code(type), address(out), o_st, o_sh, s);
  });
}

// latent_write(kv, weight, eps, positions, freqs, slots, cache, fmt, kv_scale, interleaved, factor, block_size, block_stride)
long latent_write(PyObject* const* a) {
  const at::Tensor *kv = tensor(a[0], "kv"), *w = maybe(a[1], "weight"), *pos = tensor(a[3], "positions"), *freqs = tensor(a[4], "freqs");
  const at::Tensor *slots = tensor(a[5], "slots"), *cache = tensor(a[6], "cache");
  const float eps = epsilon(number(a[2])), kv_scale = (float)number(a[8]);
  const double factor = number(a[10]);
  const long long fmt = integer(a[7]);
  const bool inter = truth(a[9]);
  if (kv->dim() != 2 || kv->size(1) != 576 || type_of(*kv) != BF16 || kv->stride(1) != 1)
    refuse("kv [n, 576] bf16 with contiguous rows: got " + shown(*kv));
  if (fmt < 0 || fmt > 2) refuse("fmt must be one of 0, 1, 2: got " + std::to_string(fmt));
  const int64_t rowb = fmt == 0 ? 656 : fmt == 1 ? 576 : 400, cd = cache->dim();
  if (cd < 2 || cd > 3 || type_of(*cache) != U8 || cache->size(cd - 1) != rowb || cache->stride(cd - 1) != 1)
    refuse("cache rows of uint8, " + std::to_string(rowb) + " bytes, [R, row] or [blocks, block_size, row]: got " + shown(*cache));
  if (fmt != 0 && !(kv_scale > 0.f)) refuse("kv_scale > 0: got " + std::to_string(kv_scale));
  line(*slots, 0, ANY, I64, "slots [n] int64");
  const int64_t n = std::min(kv->size(0), slots->size(0)), kv_st = kv->size(0) > 1 ? kv->stride(0) : 576;
  at_most(n, MAX_TOKENS, "n");
  if (n > 0) on_bytes(*kv, 2 * kv_st, 16, "kv [n, 576] bf16");
  if (n > 0 && w) on_bytes(*w, 0, 16, "weight [512]");
  if (w) line(*w, 512, 512, BF16 | F32, "weight [512] bf16 / fp32");
  line(*pos, n, ANY, I32 | I64, "positions [T] int32 / int64");
  line(*freqs, 32, 32, F64, "freqs [32] float64");
  int64_t R, bs, bstride;
  if (cd == 3) {
    R = cache->size(0) * cache->size(1);
    bs = cache->size(1);
    bstride = cache->size(0) > 1 ? cache->stride(0) : bs * rowb;
    if (bs > 1 && cache->stride(1) != rowb) refuse("cache: rows inside a block must be contiguous");
  } else {
    R = cache->size(0);
    if (R > 1 && a[12] == Py_None && cache->stride(0) != rowb) refuse("cache rows: contiguous, or with a block_stride");
    bs = a[11] == Py_None ? std::max<int64_t>(1, R) : integer(a[11]);
    bstride = a[12] == Py_None ? bs * rowb : integer(a[12]);
  }
  const int ni = as_int(n, "n"), bsi = as_int(bs, "block_size"), wf = w && type_of(*w) == F32;
  if (n > 0 && R > 0) {
    if (bs <= 0) refuse("block_size > 0: got " + std::to_string(bs));
    on_bytes(*cache, bstride, 8, "cache");
    if (bstride < bs * rowb) refuse("block_stride of " + std::to_string(bstride) + ": blocks of " + std::to_string(bs) + " rows overlap");
    // a [R, row] tensor with strides of its own says where its first row lies, its memory where the last may end
    const __int128 last = (__int128)((R - 1) / bs) * bstride + (R - 1) % bs * rowb + rowb;
    if (cd == 2 && last > (int64_t)cache->storage().nbytes() - cache->storage_offset())
      refuse("cache: " + std::to_string(R) + " rows in blocks of " + std::to_string(bs) + ", " + std::to_string(bstride) + " bytes apart, end behind its memory");
  }
  const int dev = gpu_of(*kv);
  for (const at::Tensor* t : {kv, w, pos, freqs, slots})
    if (t) same_gpu(*t, dev, "latent_write");
  if (cache->is_cuda()) same_gpu(*cache, dev, "latent_write");
  else if (!cache->is_pinned()) refuse("cache: on the GPU or in pinned host memory");      // an offloaded layer's rows
  return launch(dev, [&](void* s) {
    return f_latent_write(address(kv), kv_st, address(w), wf, eps, address(pos), type_of(*pos) == I32, (const double*)address(freqs), inter,
                          (float)factor, (const long long*)address(slots), ni, address(cache),
                          R, bsi, bstride, (int)fmt, kv_scale, s);
  });
}

template <long (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != N) return PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
  try {
    return PyLong_FromLong(F(a));
  } catch (const Raised&) {
    return nullptr;
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

#define CALLABLE(name, n) {#name, (PyCFunction)(void (*)())entry<name, n>, METH_FASTCALL, nullptr}
PyMethodDef calls[] = {CALLABLE(rms_norm, 9), CALLABLE(quant_fp8, 4), CALLABLE(linear_fp8, 5), CALLABLE(linear_quant, 6),
                       CALLABLE(rope, 8), CALLABLE(latent_write, 13)};

PyObject* load(PyObject*, PyObject* args) {
  const char* path;
  PyObject *rs, *gd;
  if (!PyArg_ParseTuple(args, "sOO", &path, &rs, &gd)) return nullptr;
  void* h = dlopen(path, RTLD_NOW | RTLD_LOCAL);
  if (!h) return PyErr_Format(PyExc_OSError, "%s", dlerror());
#define BIND(name)                                                                                   \
  f_##name = (decltype(f_##name))dlsym(h, "spmla_" #name);                                           \
  if (!f_##name) return PyErr_Format(PyExc_OSError, "%s: no spmla_" #name, path);
  BIND(rms_norm) BIND(quant_fp8) BIND(linear_fp8) BIND(rope) BIND(latent_write)
  Py_INCREF(rs);
  Py_INCREF(gd);
  raw_stream = rs;
  get_device = gd;
  PyObject* d = PyDict_New();
  for (PyMethodDef& def : calls) {
    PyObject* f = d ? PyCFunction_New(&def, nullptr) : nullptr;
    const bool ok = f && PyDict_SetItemString(d, def.ml_name, f) == 0;
    Py_XDECREF(f);
    if (!ok) {
      Py_XDECREF(d);
      return nullptr;
    }
  }
  return d;
}

PyMethodDef methods[] = {{"load", load, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) { return PyModule_Create(&module); }
