// The norm, quantization, projection, rotary, latent-row, page-table and dense attention calls on tensors: checks of shapes, types, strides and devices,
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
decltype(&::spmla_page_step) f_page_step = nullptr;
decltype(&::spmla_page_trim) f_page_trim = nullptr;
decltype(&::spmla_attn_prompt) f_attn_prompt = nullptr;
decltype(&::spmla_attn_chunk) f_attn_chunk = nullptr;
decltype(&::spmla_attn_chunk_ws_bytes) f_attn_chunk_ws_bytes = nullptr;
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

// ---- a pool of pages: table [M, W], lens [M], held [M], free [P], state [4]
struct Pool {
  const at::Tensor *table, *lens, *held, *free, *state;
  int64_t M, W, st, P;
  int bs;
};
Pool pool_of(PyObject* const* a, PyObject* block) {
  Pool p{tensor(a[0], "table"), tensor(a[1], "lens"), tensor(a[2], "held"), tensor(a[3], "free"), tensor(a[4], "state"), 0, 0, 0, 0, 0};
  if (p.table->dim() != 2) refuse("table [requests, pages of a request] int32: got " + shown(*p.table));
  p.M = p.table->size(0), p.W = p.table->size(1);
  if (p.M == 0) refuse("table: at least one request");
  at_most(p.M, 8192, "requests");
  p.st = rows(*p.table, p.M, p.W, I32, "table [requests, pages of a request] int32", true);
  line(*p.lens, p.M, p.M, I32, "lens [requests] int32");
  line(*p.held, p.M, p.M, I32, "held [requests] int32");
  line(*p.free, 0, 0x7fffffff, I32, "free [pages] int32");
  line(*p.state, 4, 4, I32, "state [4] int32");
  p.P = p.free->size(0);
  const long long bs = integer(block);
  if (bs < 1 || bs > 1 << 20) refuse("block_size of 1 to 2^20: got " + std::to_string(bs));
  p.bs = (int)bs;
  return p;
}
int gpu_with(const Pool& p, std::initializer_list<const at::Tensor*> more, const char* what) {
  const int dev = gpu_of(*p.table);
  for (const at::Tensor* t : {p.table, p.lens, p.held, p.free, p.state}) same_gpu(*t, dev, what);
  for (const at::Tensor* t : more) same_gpu(*t, dev, what);
  return dev;
}

// page_step(table, lens, held, free, state, block_size, new, start, req, positions, slots)
long page_step(PyObject* const* a) {
  const Pool p = pool_of(a, a[5]);
  const at::Tensor *fresh = tensor(a[6], "new"), *start = tensor(a[7], "start"), *req = tensor(a[8], "req");
  const at::Tensor *pos = tensor(a[9], "positions"), *slots = tensor(a[10], "slots");
  line(*fresh, p.M, p.M, I32, "new [requests] int32");
  line(*start, p.M + 1, p.M + 1, I32, "start [requests + 1] int32");
  line(*req, 0, MAX_TOKENS, I32, "req [n] int32");
  const int64_t n = req->size(0);
  line(*pos, n, n, I64, "positions [n] int64");
  line(*slots, n, n, I64, "slots [n] int64");
  const int dev = gpu_with(p, {fresh, start, req, pos, slots}, "page_step");
  return launch(dev, [&](void* s) {
    return f_page_step((const int*)address(fresh), (int)p.M, (int*)address(p.lens), (int*)address(p.held), (int*)address(p.table), p.st,
                       as_int(p.W, "W"), (int*)address(p.free), (int)p.P, (int*)address(p.state), p.bs, (int)n, (int*)address(start),
                       (int*)address(req), (long long*)address(pos), (long long*)address(slots), s);
  });
}

// page_trim(table, lens, held, free, state, block_size, keep)
long page_trim(PyObject* const* a) {
  const Pool p = pool_of(a, a[5]);
  const at::Tensor* keep = tensor(a[6], "keep");
  line(*keep, p.M, p.M, I32, "keep [requests] int32");
  const int dev = gpu_with(p, {keep}, "page_trim");
  return launch(dev, [&](void* s) {
    return f_page_trim((const int*)address(keep), (int)p.M, (int*)address(p.lens), (int*)address(p.held), (int*)address(p.table), p.st,
                       as_int(p.W, "W"), (int*)address(p.free), (int)p.P, (int*)address(p.state), p.bs, s);
  });
}

// token and head strides of x [T, H, D] with contiguous heads; 16-byte rows; written: heads that do not overlap
struct Heads {
  int64_t st, sh;
};
Heads heads(const at::Tensor& x, int64_t T, int64_t H, int64_t D, unsigned type, const char* what, bool written = false) {
  if (x.dim() != 3 || x.size(0) != T || x.size(1) != H || x.size(2) != D || type_of(x) != type)
    refuse(std::string(what) + " expected, (" + std::to_string(T) + ", " + std::to_string(H) + ", " + std::to_string(D) + "): got " + shown(x));
  const Heads s{T > 1 ? x.stride(0) : 0, H > 1 ? x.stride(1) : 0};
  if (T == 0 || H == 0 || D == 0) return s;
  if (D > 1 && x.stride(2) != 1) refuse(std::string(what) + ": contiguous heads");
  on_bytes(x, (s.st | s.sh) * 2, 16, what);
  if (written && ((T > 1 && s.st < D) || (H > 1 && s.sh < D) || (T > 1 && H > 1 && s.st < (H - 1) * s.sh + D && s.sh < (T - 1) * s.st + D)))
    refuse(std::string(what) + ": heads that do not overlap");
  return s;
}
// lse [T, H] fp32: token stride
int64_t sums(const at::Tensor* lse, int64_t T, int64_t H) { return lse ? rows(*lse, T, H, F32, "lse [T, H] fp32", true) : 0; }
int64_t starts(const at::Tensor& start) {
  line(start, 1, MAX_TOKENS, I32, "start [requests + 1] int32");
  return start.size(0) - 1;
}

// attend_prompt(q, k, v, start, scale, causal, out, lse)
long attend_prompt(PyObject* const* a) {
  const at::Tensor *q = tensor(a[0], "q"), *k = tensor(a[1], "k"), *v = tensor(a[2], "v"), *start = tensor(a[3], "start");
  const at::Tensor *out = tensor(a[6], "out"), *lse = maybe(a[7], "lse");
  const double scale = number(a[4]);
  const bool causal = truth(a[5]);
  const unsigned type = type_of(*q);
  if (q->dim() != 3 || !(type & (F16 | BF16))) refuse("q [T, H, D] fp16 / bf16: got " + shown(*q));
  if (k->dim() != 3 || v->dim() != 3) refuse("k [T, Hk, D], v [T, Hk, Dv]: got " + shown(*k) + ", " + shown(*v));
  const int64_t T = q->size(0), H = q->size(1), D = q->size(2), Hk = k->size(1), Dv = v->size(2);
  if (Hk == 0 || H % Hk) refuse("heads of q a multiple of k's: got " + std::to_string(H) + ", " + std::to_string(Hk));
  if (D == 0 || Dv == 0 || D % 8 || Dv % 8 || D > 256 || Dv > 256)
    refuse("D, Dv multiples of 8 up to 256: got " + std::to_string(D) + ", " + std::to_string(Dv));
  if (!((float)scale - (float)scale == 0.f)) refuse("scale: a finite number");
  at_most(T, MAX_TOKENS, "T");
  at_most(H, 65536, "H");
  const Heads qs = heads(*q, T, H, D, type, "q [T, H, D]"), ks = heads(*k, T, Hk, D, type, "k [T, Hk, D] of q's type");
  const Heads vs = heads(*v, T, Hk, Dv, type, "v [T, Hk, Dv] of q's type"), os = heads(*out, T, H, Dv, type, "out [T, H, Dv] of q's type", true);
  const int64_t ls = sums(lse, T, H), B = starts(*start);
  const int dev = gpu_of(*q);
  for (const at::Tensor* t : {q, k, v, start, out, lse})
    if (t) same_gpu(*t, dev, "attend_prompt");
  return launch(dev, [&](void* s) {
    return f_attn_prompt(address(q), qs.st, qs.sh, address(k), ks.st, ks.sh, address(v), vs.st, vs.sh, (const int*)address(start), (int)B,
                         (int)T, (int)H, (int)Hk, (int)D, (int)Dv, (float)scale, causal, dtype_code(type), address(out), os.st, os.sh,
                         (float*)address(lse), ls, s);
  });
}

// attend_chunk(q, cache, table, seqs, start, sm_scale, kv_scale, longest, items, out, lse, ws)
long attend_chunk(PyObject* const* a) {
  const at::Tensor *q = tensor(a[0], "q"), *cache = tensor(a[1], "cache"), *table = tensor(a[2], "block_table"), *seqs = tensor(a[3], "seq_lens");
  const at::Tensor *start = tensor(a[4], "start"), *out = tensor(a[9], "out"), *lse = maybe(a[10], "lse"), *ws = maybe(a[11], "ws");
  const double sm = number(a[5]), kvs = number(a[6]);
  const long long longest = integer(a[7]), items = integer(a[8]);
  if (q->dim() != 3 || type_of(*q) != BF16 || q->size(2) != 576) refuse("q [T, H, 576] bf16: got " + shown(*q));
  const int64_t T = q->size(0), H = q->size(1), B = starts(*start);
  at_most(T, MAX_TOKENS, "T");
  at_most(H, 65536, "H");
  const Heads qs = heads(*q, T, H, 576, BF16, "q [T, H, 576]"), os = heads(*out, T, H, 512, BF16, "out [T, H, 512] bf16", true);
  const int64_t ls = sums(lse, T, H);
  if (cache->dim() != 3 || type_of(*cache) != U8 || (cache->size(2) != 656 && cache->size(2) != 576))
    refuse("cache [blocks, block_size, 656 or 576] uint8: got " + shown(*cache));
  const int64_t blocks = cache->size(0), bs = cache->size(1), rowb = cache->size(2);
  if (bs == 0) refuse("cache: blocks of at least one row");
  if (cache->stride(2) != 1 || (bs > 1 && cache->stride(1) != rowb)) refuse("cache: rows inside a block must be contiguous");
  const int64_t bst = blocks > 1 ? cache->stride(0) : bs * rowb;
  if (bst % rowb || bst < bs * rowb) refuse("cache: blocks a whole number of rows apart that do not overlap");
  on_bytes(*cache, 0, 16, "cache");
  const int64_t stride = bst / rowb, total = blocks > 0 ? (blocks - 1) * stride + bs : 0;
  at_most(total, 0x7fffffff, "rows of the cache");
  if (table->dim() != 2) refuse("block_table [requests, columns] int32: got " + shown(*table));
  const int64_t W = table->size(1), tst = rows(*table, B, W, I32, "block_table [requests, columns] int32");
  at_most(W * bs, 0x7fffff00, "positions of a block table's row");
  line(*seqs, B, B, I32, "seq_lens [requests] int32");
  if (!((float)(sm * kvs) - (float)(sm * kvs) == 0.f)) refuse("sm_scale, kv_scale: finite numbers");
  if (longest < 0 || longest > 0x7fffffff) refuse("longest of 0 to 2^31 - 1: got " + std::to_string(longest));
  if (items < 0 || items > 65536) refuse("items of 0 to 65536: got " + std::to_string(items));
  const long long need = f_attn_chunk_ws_bytes((int)T, (int)H, (int)B, (int)rowb, (int)(longest < W * bs ? longest : W * bs), (int)items);
  if (need > 0) {
    if (!ws) refuse("ws: a workspace of " + std::to_string(need) + " bytes");
    line(*ws, need, ANY, U8, "ws uint8 (spmla_attn_chunk_ws_bytes)");
    on_bytes(*ws, 0, 16, "ws");
  }
  const int dev = gpu_of(*q);
  for (const at::Tensor* t : {q, cache, table, seqs, start, out, lse, ws})
    if (t) same_gpu(*t, dev, "attend_chunk");
  return launch(dev, [&](void* s) {
    return f_attn_chunk(address(q), qs.st, qs.sh, address(cache), total, (int)rowb, as_int(bs, "block_size"), stride,
                        (const int*)address(table), tst, (int)W, (const int*)address(seqs), (const int*)address(start), (int)B, (int)T,
                        (int)H, (float)sm, (float)kvs, (int)longest, (int)items, address(out), os.st, os.sh, (float*)address(lse), ls,
                        address(ws), ws ? ws->numel() : 0, s);
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
                       CALLABLE(rope, 8), CALLABLE(latent_write, 13), CALLABLE(page_step, 11), CALLABLE(page_trim, 7),
                       CALLABLE(attend_prompt, 8), CALLABLE(attend_chunk, 12)};

PyObject* load(PyObject*, PyObject* args) {
  const char* path;
  PyObject *rs, *gd;
  if (!PyArg_ParseTuple(args, "sOO", &path, &rs, &gd)) return nullptr;
  void* h = dlopen(path, RTLD_NOW | RTLD_LOCAL);
  if (!h) return PyErr_Format(PyExc_OSError, "%s", dlerror());
#define BIND(name)                                                                                   \
  f_##name = (decltype(f_##name))dlsym(h, "spmla_" #name);                                           \
  if (!f_##name) return PyErr_Format(PyExc_OSError, "%s: no spmla_" #name, path);
  BIND(rms_norm) BIND(quant_fp8) BIND(linear_fp8) BIND(rope) BIND(latent_write) BIND(page_step) BIND(page_trim)
  BIND(attn_prompt) BIND(attn_chunk) BIND(attn_chunk_ws_bytes)
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
