// The calls of the operators on drafted trees, from Python to their launchers: checks of the arguments, the device, the stream, the workspace.
// A call of one of them passes ten to twenty tensors; looked at from Python that takes 12 to 35 us, several times what the smaller kernels
// themselves take, and here about 2.  What the operators do and take is said in kernels.py.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <string>

namespace {

PyObject* g_error = nullptr;                     // kernels.KernelError
struct Refused {};                               // the Python error is set

[[noreturn]] void refuse(const std::string& text) {
  PyErr_SetString(g_error, text.c_str());
  throw Refused{};
}
std::string shape_text(at::IntArrayRef s) {
  std::string t = "[";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + "]";
}

// The arguments of a call, one after the other; they all have to be on one CUDA device (`device`).
struct Reader {
  PyObject* const* args;
  Py_ssize_t n, at = 0;
  const char* what;
  const at::Tensor* first = nullptr;
  bool mixed = false;
  Reader(PyObject* const* a, Py_ssize_t count, Py_ssize_t want, const char* w) : args(a), n(count), what(w) {
    if (count != want) {
      PyErr_Format(PyExc_TypeError, "%s: %zd arguments, not %zd", w, want, count);
      throw Refused{};
    }
  }
  const at::Tensor* tensor(const char* name, bool optional = false) {
    PyObject* o = args[at++];
    if (optional && o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) {
      PyErr_Format(PyExc_TypeError, "%s: %s must be a tensor", what, name);
      throw Refused{};
    }
    const at::Tensor* t = &THPVariable_Unpack(o);
    if (!first) first = t;
    mixed |= t->device() != first->device();
    return t;
  }
  long long integer() {
    const long long v = PyLong_AsLongLong(args[at++]);
    if (v == -1 && PyErr_Occurred()) throw Refused{};
    return v;
  }
  int small(const char* name) {                  // an int of C
    const long long v = integer();
    if (v < -2147483647ll || v > 2147483647ll) refuse(std::string(what) + ": " + name + "=" + std::to_string(v));
    return (int)v;
  }
  double real() {
    const double v = PyFloat_AsDouble(args[at++]);
    if (v == -1.0 && PyErr_Occurred()) throw Refused{};
    return v;
  }
  void* pointer() {
    void* p = PyLong_AsVoidPtr(args[at++]);
    if (!p && PyErr_Occurred()) throw Refused{};
    return p;
  }
  c10::DeviceIndex device() const {
    if (!first->is_cuda()) refuse("lmsf_b200 kernels run on CUDA tensors only; got a tensor on " + first->device().str());
    if (mixed) refuse(std::string(what) + ": tensors on several devices");
    return first->device().index();
  }
};

void* data(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

// A contiguous tensor of this type and shape.
void must_be(const at::Tensor* t, at::ScalarType type, std::initializer_list<int64_t> shape, const char* name) {
  if (!t) return;
  if (t->scalar_type() == type && t->sizes() == at::IntArrayRef(shape.begin(), shape.size()) && t->is_contiguous()) return;
  refuse(std::string(name) + " must be a contiguous " + (type == at::kInt ? "int32" : type == at::kLong ? "int64" : "float32") + " tensor " +
         shape_text(at::IntArrayRef(shape.begin(), shape.size())) + ", not " + c10::toString(t->scalar_type()) + " " + shape_text(t->sizes()));
}
void must_be_ints(const at::Tensor* t, std::initializer_list<int64_t> shape, const char* name) { must_be(t, at::kInt, shape, name); }
// The size of dimension d, -1 where there is none.
int64_t size_of(const at::Tensor* t, int64_t d) { return t && d < t->dim() ? t->size(d) : -1; }

// Tensors of one option: all of them or none.
void together(std::initializer_list<const at::Tensor*> ts, const char* names) {
  size_t given = 0;
  for (const at::Tensor* t : ts) given += t != nullptr;
  if (given && given != ts.size()) refuse(std::string(names) + " belong together");
}
// Whether rows of x and of y (2-dimensional, contiguous in the last dimension) share memory; columns of one buffer do not.
bool overlap(const at::Tensor& x, const at::Tensor& y) {
  if (!x.numel() || !y.numel()) return false;
  const int64_t nx = x.size(0), ny = y.size(0), wx = x.size(1) * x.element_size(), wy = y.size(1) * y.element_size();
  const int64_t px = (int64_t)x.data_ptr(), py = (int64_t)y.data_ptr(), sx = nx > 1 ? x.stride(0) * x.element_size() : wx, sy = ny > 1 ? y.stride(0) * y.element_size() : wy;
  if (px + (nx - 1) * sx + wx <= py || py + (ny - 1) * sy + wy <= px) return false;
  if (sx != sy || sx <= 0) return true;
  const int64_t d = ((py - px) % sx + sx) % sx;
  return d < wx || d + wy > sx;
}
// Whether one of n rows of `width` bytes, `stride` apart from `rows` on, lies in the bytes of y, which is contiguous.
bool rows_in(int64_t rows, int64_t n, int64_t width, int64_t stride, const at::Tensor& y) {
  const int64_t from = (int64_t)y.data_ptr(), to = from + y.numel() * y.element_size();
  if (n < 1 || width < 1 || from == to) return false;
  const int64_t before = from - rows - width;      // the first row that ends behind y's first byte
  const int64_t i = before < 0 ? 0 : stride > 0 ? before / stride + 1 : n;
  return i < n && rows + i * stride < to;
}
// The distance of rows that a kernel is given; of a single row it says nothing.
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
constexpr int64_t kMost = 1ll << 30;             // of sizes that kernels count in 32 bits, with room for what they add

int fits(int64_t v, const char* what) {
  if (v > kMost) refuse(std::string(what) + ": a size of " + std::to_string(v));
  return (int)v;
}
int dtype_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kFloat) return 0;
  if (t.scalar_type() == at::kBFloat16) return 1;
  refuse(std::string("kernels take float32 or bfloat16, not ") + c10::toString(t.scalar_type()));
}

template <typename F>
PyObject* guarded(F f) {
  try {
    return PyLong_FromLong(f());
  } catch (const Refused&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "an unknown C++ exception");
  }
  return nullptr;
}

constexpr int kMaxNodes = 256;
// Answers beside a launcher's own (0, a CUDA error above 0, -1: refused)
constexpr int kRefusedByPlain = -2, kNothing = -3;

PyObject* tree_layout(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> int {
    const char* what = "tree_layout";
    Reader r(args, n, 13, what);
    auto launch = (int (*)(void*, void*, void*, void*, void*, const void*, const void*, const void*, const void*, int, int, int, int, int, int, void*, void*))r.pointer();
    const at::Tensor *cu_q = r.tensor("cu_q"), *token_seq = r.tensor("token_seq"), *positions = r.tensor("positions"), *slots = r.tensor("slots"),
                     *mask = r.tensor("mask", true), *parents = r.tensor("parents", true), *tree_len = r.tensor("tree_len"),
                     *prefix_len = r.tensor("prefix_len"), *table = r.tensor("block_table");
    const int block_size = r.small("block_size"), window = r.small("window");
    const at::Tensor* flag = r.tensor("error_flag", true);
    const int64_t S = size_of(tree_len, 0), N = size_of(token_seq, 0);
    fits(S, what);
    fits(N, what);
    must_be_ints(tree_len, {S}, "tree_len");
    must_be_ints(prefix_len, {S}, "prefix_len");
    must_be_ints(cu_q, {S + 1}, "cu_q");
    must_be_ints(token_seq, {N}, "token_seq");
    must_be_ints(positions, {N}, "positions");
    must_be(slots, at::kLong, {N}, "tree_layout: slots");
    must_be_ints(parents, {N}, "parents");
    if (table->dim() != 2) refuse("tree_layout: the block table has one row per request");
    must_be_ints(table, {S, table->size(1)}, "block_table");
    int words = 0;
    if (mask) {
      must_be_ints(mask, {N, size_of(mask, 1)}, "tree_layout: mask");
      if (mask->size(1) < 1 || mask->size(1) > kMaxNodes / 32)
        refuse("tree_layout: a mask has 1 to " + std::to_string(kMaxNodes / 32) + " words a row, not " + std::to_string(mask->size(1)));
      words = (int)mask->size(1);
    } else if (window) {
      refuse("tree_layout: a window shows in the mask");
    }
    if (block_size < 1 || window < 0) refuse("tree_layout: block_size=" + std::to_string(block_size) + ", window=" + std::to_string(window));
    must_be_ints(flag, {1}, "error_flag");
    const c10::cuda::CUDAGuard guard(r.device());
    return launch(data(cu_q), data(token_seq), data(positions), data(slots), data(mask), data(parents), data(tree_len), data(prefix_len), data(table),
                  fits(table->size(1), what), block_size, fits(S, what), fits(N, what), words, window, data(flag), c10::cuda::getCurrentCUDAStream().stream());
  });
}


PyObject* attention_tree(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> int {
    const char* what = "attention_tree";
    Reader r(args, n, 22, what);
    // the tensor-core kernel (0: not to be used) and the other, and their workspaces in bytes
    auto tc = (int (*)(const void*, long long, const void*, long long, const void*, long long, void*, long long, const void*, long long, long long, int, const void*, int, int,
                       const void*, const void*, const void*, int, const void*, int, float, int, int, int, int, int, void*, int, void*, void*))r.pointer();
    auto plain = (int (*)(const void*, long long, const void*, long long, const void*, long long, void*, long long, const void*, long long, long long, int, const void*, int,
                          int, const void*, const void*, const void*, int, const void*, int, float, int, int, int, int, int, int, void*, int, void*))r.pointer();
    const long long tc_bytes = r.integer(), plain_bytes = r.integer();
    const int sms = r.small("sms");
    const at::Tensor *out = r.tensor("out"), *q = r.tensor("q"), *k = r.tensor("k"), *v = r.tensor("v"), *cache = r.tensor("cache"), *table = r.tensor("block_table");
    const int64_t block_size = r.integer();
    const at::Tensor *cu_q = r.tensor("cu_q"), *prefix = r.tensor("prefix_len"), *mask = r.tensor("mask");
    const double scale = r.real();
    const int64_t heads = r.integer(), kvh = r.integer(), hd = r.integer();
    const at::Tensor* positions = r.tensor("positions", true);
    const int window = r.small("window");
    const at::Tensor* flag = r.tensor("error_flag", true);
    const int64_t N = size_of(q, 0), S = size_of(prefix, 0);
    if (heads < 1 || kvh < 1 || heads % kvh) refuse("attention_tree: " + std::to_string(heads) + " query heads of " + std::to_string(kvh) + " kv heads");
    if (q->dim() != 2 || k->dim() != 2 || q->size(1) != heads * hd || out->sizes() != q->sizes() || k->size(0) != N || k->size(1) != kvh * hd || v->sizes() != k->sizes())
      refuse("attention_tree: q and out must be [rows, heads * head_dim], k and v [rows, kv heads * head_dim]");
    if (N && hd && (q->stride(1) != 1 || out->stride(1) != 1 || k->stride(1) != 1 || v->stride(1) != 1))
      refuse("attention_tree: q, k, v and out need a contiguous last dimension");
    const int code = dtype_code(*q);
    const at::ScalarType type = q->scalar_type();
    if (out->scalar_type() != type || k->scalar_type() != type || v->scalar_type() != type || cache->scalar_type() != type)
      refuse("attention_tree: q, k, v, out and the cache must share one dtype");
    if (cache->dim() != 5 || cache->size(1) != 2 || cache->size(2) != kvh || cache->size(3) != block_size || cache->size(4) != hd || !cache->is_contiguous())
      refuse("attention_tree: cache of shape " + shape_text(cache->sizes()) + " does not match [pages, 2, " + std::to_string(kvh) + ", " + std::to_string(block_size) + ", " +
             std::to_string(hd) + "]");
    if (table->dim() != 2 || mask->dim() != 2 || mask->size(1) < 1)
      refuse("attention_tree: the block table has one row per request, the mask at least a word for every row");
    must_be_ints(prefix, {S}, "prefix_len");
    must_be_ints(table, {S, table->size(1)}, "block_table");
    must_be_ints(cu_q, {S + 1}, "cu_q");
    must_be_ints(mask, {N, mask->size(1)}, "mask");
    must_be_ints(positions, {N}, "positions");
    if (window < 0 || (window && !positions)) refuse("attention_tree: a window is positive and needs positions");
    if (!std::isfinite((float)scale)) refuse("attention_tree: the scale must be a finite float32");
    if (mask->size(1) > kMost / 32 || block_size < 1 || block_size > kMost || table->size(1) > kMost / block_size || N > kMost)
      refuse("attention_tree: " + std::to_string(table->size(1)) + " pages of " + std::to_string(block_size) + " positions, " + std::to_string(mask->size(1)) + " mask words, " +
             std::to_string(N) + " rows are more than 32 bits count");
    for (const at::Tensor* t : {q, k, v})
      if (overlap(*out, *t)) refuse("attention_tree: out shares memory with q, k or v");
    if (out->numel() && rows_in((int64_t)out->data_ptr(), N, out->size(1) * out->element_size(), row_stride(*out) * out->element_size(), *cache))
      refuse("attention_tree: out shares memory with the cache");
    if (out->numel() && row_stride(*out) < out->size(1)) refuse("attention_tree: rows of out share memory");
    must_be_ints(flag, {1}, "error_flag");
    const c10::cuda::CUDAGuard guard(r.device());
    if (N == 0 || S == 0) return kNothing;
    const int64_t qs = row_stride(*q), ks = row_stride(*k), vs = row_stride(*v), os = row_stride(*out);
    const auto addresses = (uintptr_t)q->data_ptr() | (uintptr_t)k->data_ptr() | (uintptr_t)v->data_ptr() | (uintptr_t)cache->data_ptr();
    const bool on_tc = tc && code == 1 && heads / kvh <= 128 && block_size >= 8 && (block_size & (block_size - 1)) == 0 && cache->size(0) > 0 && (float)scale > 0.f &&
                       (qs | ks | vs) % 8 == 0 && std::min(qs, std::min(ks, vs)) > 0 && addresses % 16 == 0;
    const at::Tensor space = at::empty({on_tc ? tc_bytes : plain_bytes}, q->options().dtype(at::kByte));
    void* stream = c10::cuda::getCurrentCUDAStream().stream();
    const int pages = fits(cache->size(0), what), blocks = fits(table->size(1), what), words = fits(mask->size(1), what), bs = fits(block_size, what);
    if (on_tc)
      return tc(q->data_ptr(), qs, k->data_ptr(), ks, v->data_ptr(), vs, out->data_ptr(), os, cache->data_ptr(), cache->stride(0),
                cache->stride(1), pages, data(table), blocks, bs, data(cu_q), data(prefix), data(mask), words, data(positions), window, (float)scale, fits(S, what),
                fits(N, what), (int)heads, (int)kvh, (int)hd, space.data_ptr(), sms, data(flag), stream);
    const int rc = plain(q->data_ptr(), qs, k->data_ptr(), ks, v->data_ptr(), vs, out->data_ptr(), os, cache->data_ptr(),
                         cache->stride(0), cache->stride(1), pages, data(table), blocks, bs, data(cu_q), data(prefix), data(mask), words, data(positions), window, (float)scale,
                         fits(S, what), fits(N, what), (int)heads, (int)kvh, (int)hd, code, space.data_ptr(), sms, stream);
    return rc < 0 ? kRefusedByPlain : rc;
  });
}

PyObject* adjust_logits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> int {
    const char* what = "adjust_logits";
    Reader r(args, n, 19, what);
    auto launch = (int (*)(void*, long long, const void*, long long, int, int, const void*, int, const void*, long long, int, const void*, const void*, const void*, const void*,
                           const void*, const void*, const void*, const void*, int, const void*, const void*, const void*, int, const void*, const void*, int, int, void*,
                           void*))r.pointer();
    const at::Tensor *out = r.tensor("out"), *logits = r.tensor("logits"), *row_req = r.tensor("row_req", true);
    const at::Tensor *history = r.tensor("history", true), *length = r.tensor("length", true), *prompt = r.tensor("prompt length", true);
    const at::Tensor *presence = r.tensor("presence", true), *frequency = r.tensor("frequency", true), *repetition = r.tensor("repetition", true);
    const at::Tensor *tokens = r.tensor("tree tokens", true), *mask = r.tensor("tree mask", true), *cu_q = r.tensor("cu_q", true);
    const at::Tensor *b_start = r.tensor("bias start", true), *b_token = r.tensor("bias token", true), *b_value = r.tensor("bias value", true);
    const at::Tensor *bits = r.tensor("masks", true), *which = r.tensor("mask of a row", true);
    const at::Tensor* flag = r.tensor("error_flag", true);
    if (logits->dim() != 2 || logits->scalar_type() != at::kFloat || out->scalar_type() != at::kFloat || out->sizes() != logits->sizes())
      refuse("adjust_logits: logits and out must be float32 [rows, vocab]");
    const int64_t rows = logits->size(0), vocab = logits->size(1);
    const bool some = rows && vocab;
    if (some && (logits->stride(1) != 1 || out->stride(1) != 1 || (rows > 1 && (logits->stride(0) < vocab || out->stride(0) < vocab))))
      refuse("adjust_logits: logits and out need a contiguous last dimension and rows apart");
    if (some && (out->data_ptr() != logits->data_ptr() || row_stride(*out) != row_stride(*logits)) && overlap(*out, *logits))
      refuse("adjust_logits: out is logits itself or lies apart from it");
    together({history, length, prompt}, "adjust_logits: a history's tokens, lengths and prompt lengths");
    together({presence, frequency, repetition}, "adjust_logits: the three penalties");
    together({tokens, mask, cu_q}, "adjust_logits: a tree's tokens, mask and cu_q");
    together({b_start, b_token, b_value}, "adjust_logits: a bias's starts, tokens and values");
    together({bits, which}, "adjust_logits: masks and which of them a row takes");
    if ((history || tokens) && !presence) refuse("adjust_logits: occurrences are counted for penalties");
    const int64_t R = presence ? size_of(presence, 0) : b_start ? size_of(b_start, 0) - 1 : 0;
    must_be(presence, at::kFloat, {R}, "adjust_logits: presence");
    must_be(frequency, at::kFloat, {R}, "adjust_logits: frequency");
    must_be(repetition, at::kFloat, {R}, "adjust_logits: repetition");
    if (history) {
      if (history->scalar_type() != at::kInt || history->dim() != 2 || history->size(0) != R || (history->numel() && history->stride(1) != 1))
        refuse("adjust_logits: the history must be int32 [requests, width] with a contiguous last dimension");
      must_be_ints(length, {R}, "adjust_logits: the history's length");
      must_be_ints(prompt, {R}, "adjust_logits: the prompts' length");
    }
    if (tokens) {
      must_be_ints(tokens, {rows}, "adjust_logits: tree tokens");
      must_be_ints(mask, {rows, size_of(mask, 1)}, "adjust_logits: tree mask");
      must_be_ints(cu_q, {R + 1}, "adjust_logits: cu_q");
    }
    if (b_start) {
      must_be_ints(b_start, {R + 1}, "adjust_logits: bias start");
      must_be_ints(b_token, {size_of(b_token, 0)}, "adjust_logits: bias token");
      must_be(b_value, at::kFloat, {b_token->size(0)}, "adjust_logits: bias value");
    }
    const int64_t words = (vocab + 31) / 32;
    if (bits) {
      must_be_ints(bits, {size_of(bits, 0), words}, "adjust_logits: masks");
      must_be_ints(which, {rows}, "adjust_logits: mask of a row");
    }
    if (!row_req && R && R != rows) refuse("adjust_logits: options of " + std::to_string(R) + " requests for " + std::to_string(rows) + " rows need row_req");
    must_be_ints(row_req, {rows}, "adjust_logits: row_req");
    must_be_ints(flag, {1}, "error_flag");
    const c10::cuda::CUDAGuard guard(r.device());
    if (!some) return kNothing;
    return launch(out->data_ptr(), std::max(out->stride(0), vocab), logits->data_ptr(), std::max(logits->stride(0), vocab), fits(rows, what), fits(vocab, what), data(row_req),
                  presence || b_start ? fits(R, what) : -1, data(history), history ? history->stride(0) : 0, history ? fits(history->size(1), what) : 0, data(length), data(prompt), data(presence),
                  data(frequency), data(repetition), data(tokens), data(mask), data(cu_q), mask ? fits(mask->size(1), what) : 0, data(b_start), data(b_token), data(b_value),
                  b_token ? fits(b_token->size(0), what) : 0, data(bits), data(which), bits ? fits(bits->size(0), what) : 0, bits ? fits(words, what) : 0, data(flag),
                  c10::cuda::getCurrentCUDAStream().stream());
  });
}

PyObject* tree_accept(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> int {
    const char* what = "tree_accept";
    Reader r(args, n, 15, what);
    auto launch = (int (*)(void*, void*, void*, void*, const void*, const void*, const void*, const void*, const void*, int, int, int, const void*, const void*, const void*,
                           long long, long long, long long, long long, void*, int, int, int, int, int, void*, void*))r.pointer();
    const at::Tensor *n_kept = r.tensor("n_kept"), *path = r.tensor("path"), *next = r.tensor("next_token"), *new_len = r.tensor("new_len"), *target = r.tensor("target"),
                     *tokens = r.tensor("tokens"), *parents = r.tensor("parents"), *cu_q = r.tensor("cu_q"), *prefix = r.tensor("prefix_len");
    const at::Tensor *slots = r.tensor("slots", true), *k = r.tensor("k", true), *v = r.tensor("v", true), *cache = r.tensor("cache", true);
    const at::Tensor* flag = r.tensor("error_flag", true);
    const int64_t S = size_of(prefix, 0), N = size_of(target, 0);
    if (path->dim() != 2 || path->size(0) != S || path->size(1) < 1 || path->size(1) > kMaxNodes)
      refuse("tree_accept: the path must be int32 [requests, 1 to " + std::to_string(kMaxNodes) + "]");
    must_be_ints(prefix, {S}, "prefix_len");
    must_be_ints(n_kept, {S}, "n_kept");
    must_be_ints(path, {S, path->size(1)}, "path");
    must_be_ints(next, {S}, "next_token");
    must_be_ints(new_len, {S}, "new_len");
    must_be_ints(target, {N}, "target");
    must_be_ints(tokens, {N}, "tokens");
    must_be_ints(parents, {N}, "parents");
    must_be_ints(cu_q, {S + 1}, "cu_q");
    long long strides[4] = {0, 0, 0, 0};
    int sizes[5] = {0, 0, 0, 0, 0};
    bool copy = false;
    if (slots || k || v || cache) {
      if (!slots || !k || !v || !cache) refuse("tree_accept: slots, k, v and the cache belong together");
      if (cache->dim() != 6 || cache->size(2) != 2 || !cache->is_contiguous())
        refuse("tree_accept: the cache must be contiguous [calls, pages, 2, kv heads, block_size, head_dim]");
      dtype_code(*cache);
      must_be(slots, at::kLong, {N}, "tree_accept: slots");
      const int64_t width = cache->size(3) * cache->size(5), size = cache->element_size();
      for (const at::Tensor* t : {k, v})
        if (t->scalar_type() != cache->scalar_type() || t->dim() != 3 || t->size(0) != cache->size(0) || t->size(1) != N || t->size(2) != width ||
            (t->numel() && t->stride(2) != 1))
          refuse("tree_accept: k and v must be [calls, rows, kv heads * head_dim] of the cache's dtype with a contiguous last dimension");
      copy = cache->numel() && N;
      if (copy) {
        for (const at::Tensor* t : {k, v})
          for (int64_t c = 0; c < t->size(0); ++c)
            if (rows_in((int64_t)t->data_ptr() + c * t->stride(0) * size, N, width * size, t->stride(1) * size, *cache))
              refuse("tree_accept: k and v lie apart from the cache");
        strides[0] = k->stride(0) * size; strides[1] = k->stride(1) * size; strides[2] = v->stride(0) * size; strides[3] = v->stride(1) * size;
        sizes[0] = fits(cache->size(0), what); sizes[1] = fits(cache->size(1), what); sizes[2] = fits(cache->size(3), what);
        sizes[3] = fits(cache->size(4), what); sizes[4] = fits(cache->size(5) * size, what);
      }
    }
    must_be_ints(flag, {1}, "error_flag");
    const c10::cuda::CUDAGuard guard(r.device());
    return launch(data(n_kept), data(path), data(next), data(new_len), data(target), data(tokens), data(parents), data(cu_q), data(prefix), fits(S, what), fits(N, what),
                  (int)path->size(1), copy ? data(slots) : nullptr, copy ? data(k) : nullptr, copy ? data(v) : nullptr, strides[0], strides[1], strides[2], strides[3],
                  copy ? data(cache) : nullptr, sizes[0], sizes[1], sizes[2], sizes[3], sizes[4], data(flag), c10::cuda::getCurrentCUDAStream().stream());
  });
}

PyObject* set_error(PyObject*, PyObject* type) {
  Py_XINCREF(type);
  Py_XSETREF(g_error, type);
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"tree_layout", (PyCFunction)(void (*)(void))tree_layout, METH_FASTCALL, nullptr},
    {"attention_tree", (PyCFunction)(void (*)(void))attention_tree, METH_FASTCALL, nullptr},
    {"adjust_logits", (PyCFunction)(void (*)(void))adjust_logits, METH_FASTCALL, nullptr},
    {"tree_accept", (PyCFunction)(void (*)(void))tree_accept, METH_FASTCALL, nullptr},
    {"set_error", set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "lmsf_tree_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_lmsf_tree_calls(void) { return PyModule_Create(&g_module); }
