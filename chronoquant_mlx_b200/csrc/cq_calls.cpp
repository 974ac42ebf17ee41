// cq_calls.cpp -- the Python entry points of the sparse-attention and rotation
// operators in C++: argument checks, output allocation, stream lookup and the
// call of the C library in one step.  A decode step's kernels run for 3 to 10 us;
// checked in Python and called through ctypes such a call took 11 to 18 us of
// host time, from here 5.  Python's lock is given up once the arguments are read
// (allocations and launches may wait).  The module holds no kernels and keeps
// nothing between calls; the C functions come from the library that load() is given.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <exception>
#include <stdexcept>
#include <string>

#include "../../include/chronoquant_b200.h"

namespace {

struct Library {
  decltype(&cq_last_error) last_error = nullptr;
  decltype(&cq_qk_norm_rope_rows) rope = nullptr;
  decltype(&cq_block_bounds) bounds = nullptr;
  decltype(&cq_block_bounds_read) bounds_read = nullptr;
  decltype(&cq_block_select) select = nullptr;
  decltype(&cq_block_select_workspace) select_ws = nullptr;
  decltype(&cq_sparse_attention) sparse = nullptr;
  decltype(&cq_sparse_attention_workspace) sparse_ws = nullptr;
} L;
PyObject *g_cuda_error = nullptr;  // CudaLibError

// What a check throws: the Python exception to raise.
struct Refused {
  PyObject *type;
  std::string text;
};
[[noreturn]] void refuse(PyObject *type, std::string text) { throw Refused{type, std::move(text)}; }
void require(bool ok, const char *text) {
  if (!ok) refuse(PyExc_ValueError, text);
}

void check(int status, const char *what) {
  if (status == CQ_OK) return;
  const char *m = L.last_error();
  PyObject *type = status == CQ_ERR_INVALID || status == CQ_ERR_WORKSPACE ? PyExc_ValueError
                   : status == CQ_ERR_UNSUPPORTED                         ? PyExc_NotImplementedError
                                                                          : g_cuda_error;
  refuse(type, std::string(what) + ": " + (m ? m : ""));
}

const at::Tensor &tensor(PyObject *o, const char *what) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(what) + " must be a tensor");
  return THPVariable_Unpack(o);
}
long long integer(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused{nullptr, ""};  // its own exception
  return v;
}
int32_t int32(PyObject *o, const char *what) {
  const long long v = integer(o);
  if (v < INT32_MIN || v > INT32_MAX) refuse(PyExc_ValueError, std::string(what) + " is out of range");
  return (int32_t)v;
}
bool truth(PyObject *o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Refused{nullptr, ""};
  return v != 0;
}
double real(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refused{nullptr, ""};
  return v;
}
// Python's lock given up from here to lock() or the scope's end: no call of Python's API meanwhile.
struct Unlocked {
  PyThreadState *state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked &) = delete;
  ~Unlocked() { lock(); }
  void lock() {
    if (state) PyEval_RestoreThread(state);
    state = nullptr;
  }
};

std::string shape_of(const at::Tensor &t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

// The stream of `t`'s device and, where another device is current, that device for the call.
struct Launch {
  c10::cuda::OptionalCUDAGuard guard;
  void *stream;
  explicit Launch(const at::Tensor &t) {
    const auto dev = t.device();
    if (dev.index() != c10::cuda::current_device()) guard.set_device(dev);
    stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  }
};

// The id of the capture that records the stream, 0 where it runs.
unsigned long long capture_id(void *stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo((cudaStream_t)stream, &status, &id));
  return status == cudaStreamCaptureStatusActive ? id : 0;
}

// Queries [B, Hq, Tq, D] of a cache of H kv-heads on `device`, holding T tokens.
struct Queries {
  at::Tensor t;
  int dtype;
  int32_t Hq, S;
  int64_t sb, sh, sq;
};
Queries queries(const at::Tensor &q, int64_t B, int64_t H, int64_t D, int64_t T, c10::Device device, const char *what) {
  const std::string w(what);
  if (q.dim() != 4 || q.size(0) != B || q.size(3) != D)
    refuse(PyExc_ValueError, w + ": queries must be [" + std::to_string(B) + ", Hq, Tq, " + std::to_string(D) +
                                 "], got " + shape_of(q));
  if (q.device() != device)
    refuse(PyExc_ValueError, w + ": queries on " + q.device().str() + ", the cache on " + device.str() +
                                 " (CUDA tensors only, no CPU fallback)");
  Queries r;
  if (q.scalar_type() == at::kHalf)
    r.dtype = CQ_F16;
  else if (q.scalar_type() == at::kBFloat16)
    r.dtype = CQ_BF16;
  else
    refuse(PyExc_TypeError, w + ": queries must be float16 or bfloat16");
  const int64_t Hq = q.size(1), S = q.size(2);
  if (Hq == 0 || Hq % H || Hq > INT32_MAX)
    refuse(PyExc_ValueError, w + ": " + std::to_string(Hq) + " query heads are no multiple of " + std::to_string(H) +
                                 " kv-heads");
  if (S < 1 || S > T || S > INT32_MAX)
    refuse(PyExc_ValueError, w + ": " + std::to_string(S) + " query tokens, " + std::to_string(T) + " tokens cached");
  r.t = q.stride(3) == 1 || D == 1 ? q : q.contiguous();
  r.Hq = (int32_t)Hq;
  r.S = (int32_t)S;
  r.sb = r.t.stride(0);
  r.sh = r.t.stride(1);
  r.sq = r.t.stride(2);
  return r;
}

const at::Tensor *tensor_or_none(PyObject *o, const char *what) { return o == Py_None ? nullptr : &tensor(o, what); }

at::Tensor starts_of(const at::Tensor *given, int64_t B, c10::Device device, const char *what) {
  if (!given) return {};
  const at::Tensor &s = *given;
  if (s.scalar_type() != at::kLong || s.dim() != 1 || s.size(0) != B || s.device() != device)
    refuse(PyExc_ValueError, std::string(what) + ": starts must be int64 [" + std::to_string(B) + "] on " +
                                 device.str() + ", got " + shape_of(s) + " on " + s.device().str());
  return s.contiguous();
}
const int64_t *starts_ptr(const at::Tensor &s) { return s.defined() ? s.const_data_ptr<int64_t>() : nullptr; }

// An uninitialised contiguous tensor: torch's own CUDA allocation, without its dispatcher's way there.
at::Tensor empty(at::IntArrayRef size, at::ScalarType type, c10::Device device) {
  return at::detail::empty_cuda(size, type, device, c10::nullopt);
}

PyObject *pair(at::Tensor a, at::Tensor b) {
  PyObject *x = THPVariable_Wrap(std::move(a)), *y = x ? THPVariable_Wrap(std::move(b)) : nullptr;
  if (!y) {
    Py_XDECREF(x);
    throw Refused{nullptr, ""};
  }
  PyObject *t = PyTuple_New(2);
  if (!t) {
    Py_DECREF(x);
    Py_DECREF(y);
    throw Refused{nullptr, ""};
  }
  PyTuple_SET_ITEM(t, 0, x);
  PyTuple_SET_ITEM(t, 1, y);
  return t;
}

// Runs f(args); no exception leaves it.
template <class F>
PyObject *guarded(PyObject *const *args, Py_ssize_t n, Py_ssize_t want, F f) {
  try {
    if (n != want) refuse(PyExc_TypeError, "wrong number of arguments");
    if (!L.last_error) refuse(PyExc_ImportError, "the CUDA library is not loaded");
    return f(args);
  } catch (const Refused &e) {
    if (e.type) PyErr_SetString(e.type, e.text.c_str());
  } catch (const c10::Error &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// qk_norm_rope(qkv, Hq, Hkv, inv_freq, positions, q_weight, k_weight, eps, adjacent) -> (q, k)
PyObject *qk_norm_rope(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded(args, n, 9, [](PyObject *const *a) {
    const at::Tensor &qkv_in = tensor(a[0], "qkv");
    const int32_t Hq = int32(a[1], "n_q_heads"), Hkv = int32(a[2], "n_kv_heads");
    const at::Tensor &f_in = tensor(a[3], "inv_freq"), &p_in = tensor(a[4], "positions");
    const at::Tensor *w_in[2] = {tensor_or_none(a[5], "a norm weight"), tensor_or_none(a[6], "a norm weight")};
    const float eps = (float)real(a[7]);
    const int32_t adjacent = truth(a[8]);
    Unlocked unlocked;
    if (qkv_in.dim() != 3)
      refuse(PyExc_ValueError, "qk_norm_rope: qkv must be [B, S, (Hq + 2 Hkv) * D], got " + shape_of(qkv_in));
    const int64_t B = qkv_in.size(0), S = qkv_in.size(1), width = qkv_in.size(2);
    const int64_t heads = (int64_t)Hq + 2 * (int64_t)Hkv;
    if (Hq < 1 || Hkv < 1 || width == 0 || width % heads || B > INT32_MAX || S > INT32_MAX)
      refuse(PyExc_ValueError, "qk_norm_rope: rows of " + std::to_string(width) + " do not hold " + std::to_string(Hq) +
                                   " + 2 * " + std::to_string(Hkv) + " heads");
    const int64_t D = width / heads;
    if (!qkv_in.is_cuda())
      refuse(PyExc_ValueError, "qk_norm_rope computes on CUDA tensors only (no CPU fallback); got a tensor on " +
                                   qkv_in.device().str());
    const auto st = qkv_in.scalar_type();
    const auto dev = qkv_in.device();
    if (st != at::kHalf && st != at::kBFloat16 && st != at::kFloat)
      refuse(PyExc_TypeError, "qk_norm_rope: expected float16, bfloat16 or float32");
    const int dt = st == at::kHalf ? CQ_F16 : st == at::kBFloat16 ? CQ_BF16 : CQ_F32;
    if (f_in.scalar_type() != at::kFloat || f_in.dim() != 1 || f_in.device() != dev)
      refuse(PyExc_ValueError, "qk_norm_rope: inv_freq must be fp32 [rot / 2] on " + dev.str());
    const int64_t half = f_in.size(0);
    if (2 * half > D)
      refuse(PyExc_ValueError, "qk_norm_rope: " + std::to_string(half) + " frequencies rotate more than " +
                                   std::to_string(D) + " channels");
    if (p_in.scalar_type() != at::kLong || p_in.device() != dev)
      refuse(PyExc_ValueError, "qk_norm_rope: positions must be int64 on " + dev.str());
    if (!w_in[0] != !w_in[1])
      refuse(PyExc_ValueError, "qk_norm_rope: give both norm weights or neither");
    at::Tensor w[2];
    if (w_in[0])
      for (int i = 0; i < 2; ++i) {
        const at::Tensor &x = *w_in[i];
        if (x.dim() != 1 || x.size(0) != D || x.scalar_type() != st || x.device() != dev)
          refuse(PyExc_ValueError, "qk_norm_rope: norm weights must be of qkv's type, [" + std::to_string(D) + "], on " +
                                       dev.str());
        w[i] = x.contiguous();
      }
    const bool full = p_in.dim() == 2 && p_in.size(0) == B && p_in.size(1) == S;
    const at::Tensor pos = full ? p_in : p_in.expand({B, S});
    const at::Tensor qkv = qkv_in.stride(2) == 1 ? qkv_in : qkv_in.contiguous(), f = f_in.contiguous();
    at::Tensor q = empty({B, Hq, S, D}, st, dev), k = empty({B, Hkv, S, D}, st, dev);
    const Launch at_(qkv);
    check(L.rope(qkv.const_data_ptr(), qkv.stride(0), qkv.stride(1), (int32_t)B, (int32_t)S, Hq, Hkv, (int32_t)D,
                 (int32_t)(2 * half), adjacent, w[0].defined() ? w[0].const_data_ptr() : nullptr,
                 w[1].defined() ? w[1].const_data_ptr() : nullptr, f.const_data_ptr<float>(),
                 pos.const_data_ptr<int64_t>(), pos.stride(0), pos.stride(1), eps, q.mutable_data_ptr(),
                 k.mutable_data_ptr(), dt, at_.stream),
          "qk_norm_rope");
    unlocked.lock();
    return pair(std::move(q), std::move(k));
  });
}

// A cache's index as Python holds it: codes int8 [B, H, cap, 2, D], scales fp32 [B, H, cap].
struct Index {
  const at::Tensor &codes, &scales;
  int64_t B, H, cap, D;
  Index(PyObject *c, PyObject *s) : codes(tensor(c, "codes")), scales(tensor(s, "scales")) {
    require(codes.dim() == 5 && codes.scalar_type() == at::kChar && codes.is_contiguous() && scales.dim() == 3 &&
                scales.scalar_type() == at::kFloat && scales.is_contiguous() &&
                scales.sizes() == codes.sizes().slice(0, 3) && codes.size(3) == 2 && codes.is_cuda() &&
                scales.device() == codes.device(),
            "the block index's tensors were replaced");
    B = codes.size(0);
    H = codes.size(1);
    cap = codes.size(2);
    D = codes.size(4);
  }
};

// block_bounds(descriptor, t0, T, block_tokens, codes, scales) -> the id of the capture that recorded it, 0: it runs
PyObject *block_bounds(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded(args, n, 6, [](PyObject *const *a) {
    const Index ix(a[4], a[5]);
    const cq_paged_cache cache = *(const cq_paged_cache *)integer(a[0]);
    const int64_t t0 = integer(a[1]), T = integer(a[2]);
    const int32_t bt = int32(a[3], "block_tokens");
    Unlocked unlocked;
    const Launch at_(ix.codes);
    check(L.bounds(&cache, t0, T, bt, (int8_t *)ix.codes.mutable_data_ptr(), ix.scales.mutable_data_ptr<float>(),
                   ix.cap, at_.stream),
          "BlockIndex.update");
    const unsigned long long id = capture_id(at_.stream);
    unlocked.lock();
    return PyLong_FromUnsignedLongLong(id);
  });
}

// capture_of(codes) -> the id of the capture that records the stream of the index's device, 0 where it runs
PyObject *capture_of(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded(args, n, 1, [](PyObject *const *a) {
    const Launch at_(tensor(a[0], "codes"));  // nothing here waits
    return PyLong_FromUnsignedLongLong(capture_id(at_.stream));
  });
}

// block_bounds_read(codes, scales, first, n) -> fp32 [B, H, n, 2, D]
PyObject *block_bounds_read(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded(args, n, 4, [](PyObject *const *a) {
    const Index ix(a[0], a[1]);
    const int64_t first = integer(a[2]), m = integer(a[3]);
    Unlocked unlocked;
    at::Tensor out = empty({ix.B, ix.H, m, 2, ix.D}, at::kFloat, ix.codes.device());
    const Launch at_(ix.codes);
    check(L.bounds_read((const int8_t *)ix.codes.const_data_ptr(), ix.scales.const_data_ptr<float>(), ix.B * ix.H,
                        ix.cap, first, m, (int32_t)ix.D, out.mutable_data_ptr<float>(), at_.stream),
          "BlockIndex.bounds");
    unlocked.lock();
    return THPVariable_Wrap(std::move(out));
  });
}

// Scores of a selection held at once.  A chunk of queries with more of them (4 bytes a query token, kv-head and
// block: 8192 queries over a million tokens would ask for 4.3 GB) is listed by parts.  1 GB, because parts cost a
// little: 2048 queries x 16384 blocks x 8 units take 1914 us at once, 2205 us in four parts of 256 MB.
constexpr size_t kScoreBytes = (size_t)1 << 30;

// block_select(codes, scales, block_tokens, T, queries, top, first, recent, starts, want_scores)
PyObject *block_select(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded(args, n, 10, [](PyObject *const *a) {
    const Index ix(a[0], a[1]);
    const int32_t bt = int32(a[2], "block_tokens"), top = int32(a[5], "top"), first = int32(a[6], "first"),
                  recent = int32(a[7], "recent");
    const int64_t T = integer(a[3]);
    const at::Tensor &q_in = tensor(a[4], "queries"), *starts_in = tensor_or_none(a[8], "starts");
    const bool want = truth(a[9]);
    Unlocked unlocked;
    if (top < 1 || top > 4096 || first < 0 || recent < 0 || (int64_t)first + recent > top)
      refuse(PyExc_ValueError, "select: need 1 <= top <= 4096 and first + recent <= top, got top=" +
                                   std::to_string(top) + ", first=" + std::to_string(first) +
                                   ", recent=" + std::to_string(recent));
    const auto dev = ix.codes.device();
    const Queries q = queries(q_in, ix.B, ix.H, ix.D, T, dev, "select");
    const at::Tensor starts = starts_of(starts_in, ix.B, dev, "select");
    const Launch at_(ix.codes);
    at::Tensor blocks = empty({ix.B, ix.H, q.S, top}, at::kInt, dev), scores, ws;
    if (want) scores = empty({ix.B, ix.H, q.S, top}, at::kFloat, dev);
    // n query tokens from token i on, of a sequence that ends with the last of them
    const auto list = [&](int32_t i, int32_t n, at::Tensor &to, at::Tensor &to_scores) {
      const int64_t T_n = T - (q.S - i - n);
      size_t need = 0;
      check(L.select_ws((int32_t)ix.B, (int32_t)ix.H, (int32_t)ix.D, q.Hq, n, T_n, bt, &need), "select");
      if (need > kScoreBytes && n > 1) return need;
      if (need && (!ws.defined() || (size_t)ws.numel() < need)) ws = empty({(int64_t)need}, at::kByte, dev);
      check(L.select((const int8_t *)ix.codes.const_data_ptr(), ix.scales.const_data_ptr<float>(), ix.cap, bt,
                     (int32_t)ix.B, (int32_t)ix.H, (int32_t)ix.D, T_n, nullptr,
                     (const char *)q.t.const_data_ptr() + 2 * (int64_t)i * q.sq, q.dtype, q.Hq, n, q.sb, q.sh, q.sq,
                     starts_ptr(starts), first, recent, top, to.mutable_data_ptr<int32_t>(),
                     want ? to_scores.mutable_data_ptr<float>() : nullptr, need ? ws.mutable_data_ptr() : nullptr, need,
                     at_.stream),
            "select");
      return (size_t)0;
    };
    if (const size_t need = list(0, q.S, blocks, scores)) {
      const size_t token = need / q.S;  // bytes of a query token's scores
      const int32_t fit = (int32_t)std::max<size_t>(1, kScoreBytes / token), parts = (q.S - 1) / fit + 1;
      const int32_t most = (q.S - 1) / parts + 1;  // even parts: at most `fit` tokens
      ws = empty({(int64_t)(token * most)}, at::kByte, dev);
      for (int32_t i = 0, n; i < q.S; i += n) {
        n = std::min(most, q.S - i);
        at::Tensor part = empty({ix.B, ix.H, n, top}, at::kInt, dev), part_scores;
        if (want) part_scores = empty({ix.B, ix.H, n, top}, at::kFloat, dev);
        list(i, n, part, part_scores);
        blocks.narrow(2, i, n).copy_(part);
        if (want) scores.narrow(2, i, n).copy_(part_scores);
      }
    }
    unlocked.lock();
    return want ? pair(std::move(blocks), std::move(scores)) : THPVariable_Wrap(std::move(blocks));
  });
}

// sparse_attention(descriptor, pool, T, queries, scale, blocks, block_tokens, starts, want_lse); pool: the
// store's page buffer, whose device is the cache's
PyObject *sparse_attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded(args, n, 9, [](PyObject *const *a) {
    const char *what = "chronoquant_sparse_sdpa";
    const cq_paged_cache cache = *(const cq_paged_cache *)integer(a[0]);
    const at::Tensor &pool = tensor(a[1], "the page pool"), &q_in = tensor(a[3], "queries"),
                     &b_in = tensor(a[5], "blocks"), *starts_in = tensor_or_none(a[7], "starts");
    const int64_t T = integer(a[2]), bt = integer(a[6]), B = cache.batch, H = cache.kv_heads, D = cache.head_dim;
    const float scale = (float)real(a[4]);
    const bool want = truth(a[8]);
    Unlocked unlocked;
    const auto dev = pool.device();
    const Queries q = queries(q_in, B, H, D, T, dev, what);
    if (b_in.dim() != 4 || b_in.size(0) != B || b_in.size(1) != H || b_in.size(2) != q.S ||
        b_in.scalar_type() != at::kInt)
      refuse(PyExc_ValueError, std::string(what) + ": blocks must be int32 [" + std::to_string(B) + ", " +
                                   std::to_string(H) + ", " + std::to_string(q.S) + ", n], got " + shape_of(b_in));
    if (b_in.device() != dev)
      refuse(PyExc_ValueError, std::string(what) + ": blocks on " + b_in.device().str() + ", the cache on " + dev.str());
    const int64_t top = b_in.size(3);
    if (top < 1 || top > 4096)
      refuse(PyExc_ValueError, std::string(what) + ": lists of 1 to 4096 blocks, got " + std::to_string(top));
    if (bt < 16 || bt % 16 || bt > (1 << 30))
      refuse(PyExc_ValueError, "block_tokens must be a positive multiple of 16, got " + std::to_string(bt));
    const at::Tensor starts = starts_of(starts_in, B, dev, what), blocks = b_in.contiguous();
    at::Tensor out, lse, ws;
    out = empty({B, q.Hq, q.S, D}, want ? at::kFloat : q.t.scalar_type(), dev);
    if (want) lse = empty({B, q.Hq, q.S}, at::kFloat, dev);
    const Launch at_(pool);
    size_t need = 0;
    check(L.sparse_ws(&cache, T, q.Hq, q.S, (int32_t)top, (int32_t)bt, &need), what);
    if (need) ws = empty({(int64_t)need}, at::kByte, dev);
    check(L.sparse(&cache, T, nullptr, q.t.const_data_ptr(), q.dtype, q.Hq, q.S, q.sb, q.sh, q.sq, scale,
                   starts_ptr(starts), blocks.const_data_ptr<int32_t>(), (int32_t)top, (int32_t)bt,
                   out.mutable_data_ptr(), want ? CQ_F32 : q.dtype, want ? lse.mutable_data_ptr<float>() : nullptr,
                   need ? ws.mutable_data_ptr() : nullptr, need, at_.stream),
          what);
    unlocked.lock();
    return want ? pair(std::move(out), std::move(lse)) : THPVariable_Wrap(std::move(out));
  });
}

// load(path, error_class): take the C functions from the library at `path` and raise its CUDA errors as `error_class`
PyObject *load(PyObject *, PyObject *args) {
  const char *path;
  PyObject *error;
  if (!PyArg_ParseTuple(args, "sO", &path, &error)) return nullptr;
  void *h = dlopen(path, RTLD_NOW | RTLD_LOCAL);
  if (!h) {
    PyErr_SetString(PyExc_ImportError, dlerror());
    return nullptr;
  }
  Library l;
  bool ok = true;
  auto get = [&](auto &fn, const char *name) {
    fn = (std::decay_t<decltype(fn)>)dlsym(h, name);
    ok = ok && fn;
  };
  get(l.last_error, "cq_last_error");
  get(l.rope, "cq_qk_norm_rope_rows");
  get(l.bounds, "cq_block_bounds");
  get(l.bounds_read, "cq_block_bounds_read");
  get(l.select, "cq_block_select");
  get(l.select_ws, "cq_block_select_workspace");
  get(l.sparse, "cq_sparse_attention");
  get(l.sparse_ws, "cq_sparse_attention_workspace");
  if (!ok) {
    PyErr_Format(PyExc_ImportError, "%s lacks functions of this build", path);
    return nullptr;
  }
  L = l;
  Py_INCREF(error);
  Py_XDECREF(g_cuda_error);
  g_cuda_error = error;
  Py_RETURN_NONE;
}

#define FAST(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(qk_norm_rope), FAST(block_bounds),     FAST(block_bounds_read),
                         FAST(capture_of),   FAST(block_select),     FAST(sparse_attention), {"load", load, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
