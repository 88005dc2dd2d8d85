// Call marshalling for the Python entry points: tensor checks, argument structs
// and output allocation in one native call instead of ~60 Python-level ones.
//
// Bounds: small calls are limited by the host.  Through ctypes, filling an
// argument struct, the per-tensor checks and the stream lookup took 12-15 us
// of a 19 us forward ([1, 512, 16, 64], 7 us of GPU work) and of each call of
// an append + decode step.
//
// Every function takes the plain case only: exact torch.Tensor objects with
// storage on the current device, matching dtypes, shapes and strides the
// kernels address as they are, index tensors already int32 (int64 for slots),
// no dispatch mode.  Anything else returns None before any work, and the
// Python path, which converts, copies or raises, takes the call.  Otherwise
// the result is the outputs, or the library's negative status for the caller
// to raise.  Nothing is kept between calls except the library's entry points.
//
// The norm-and-rotation and linear-attention training calls put their own nodes
// into the autograd graph: a Python Function's backward runs in the engine's thread
// and waits there for the interpreter lock, ~50 us of a ~110 us step whose GPU work
// took 77 us.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <ATen/ATen.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>

#include <climits>
#include <cmath>
#include <memory>
#include <mutex>

#include "fa355.h"

namespace {

struct Entries {
  decltype(&fa_fwd) fwd;
  decltype(&fa_decode_workspace_bytes) decode_workspace;
  decltype(&fa_paged_decode) decode;
  decltype(&fa_paged_prefill_num_splits) paged_splits;
  decltype(&fa_paged_prefill_splitkv_workspace_bytes) paged_workspace;
  decltype(&fa_paged_prefill_splitkv) paged;
  decltype(&fa_reshape_and_cache) cache_write;
  decltype(&fa_norm_rope) norm_rope;
  decltype(&fa_norm_rope_and_cache) norm_rope_cache;
  decltype(&fa_linear_fwd_workspace_bytes) linear_workspace;
  decltype(&fa_linear_fwd) linear_fwd;
  decltype(&fa_linear_decode) linear_decode;
  decltype(&fa_norm_rope_bwd_workspace_bytes) norm_rope_bwd_workspace;
  decltype(&fa_norm_rope_bwd) norm_rope_bwd;
  decltype(&fa_linear_bwd_workspace_bytes) linear_bwd_workspace;
  decltype(&fa_linear_bwd) linear_bwd;
} lib;

struct Call {
  int device;
  void* stream;
};

// A plain tensor on the call's device, or nullptr.
const at::Tensor* plain(PyObject* o, const Call& c, int64_t dim) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.dim() != dim || t.get_device() != c.device ||
      t.layout() != at::kStrided || !t.has_storage() || t.numel() == 0)
    return nullptr;
  return &t;
}

// The kernels can address it as it is: contiguous last dimension, 16-byte
// aligned, other strides multiples of 8 elements.
bool rows_ready(const at::Tensor& t) {
  const auto size = t.sizes(), stride = t.strides();
  const int64_t n = t.dim();
  if (stride[n - 1] != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) return false;
  for (int64_t i = 0; i + 1 < n; ++i)
    if (size[i] > 1 && (stride[i] % 8 != 0 || stride[i] < 0)) return false;
  return true;
}

template <size_t N>
void set_strides(int64_t (&dst)[N], const at::Tensor& t) {
  for (size_t i = 0; i < N; ++i) dst[i] = t.size(i) == 1 ? 0 : t.stride(i);
}

bool half_code(const at::Tensor& t, int32_t* code) {
  if (t.scalar_type() == at::kHalf)
    *code = FA_DTYPE_F16;
  else if (t.scalar_type() == at::kBFloat16)
    *code = FA_DTYPE_BF16;
  else
    return false;
  return true;
}

bool fits(int64_t v) { return v <= INT_MAX; }

// int32 tensor of `dim` dimensions whose rows are contiguous.
bool index_ready(const at::Tensor* t) {
  return t && t->scalar_type() == at::kInt && t->is_contiguous();
}

bool call_of(PyObject* device, PyObject* stream, Call* c) {
  if (c10::impl::TorchDispatchModeTLS::any_modes_set()) return false;
  c->device = (int)PyLong_AsLong(device);
  c->stream = PyLong_AsVoidPtr(stream);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool number(PyObject* o, float* out) {
  if (!PyFloat_Check(o) && !PyLong_Check(o)) return false;
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  *out = (float)v;
  return true;
}

bool integer(PyObject* o, int64_t* out) {
  if (!PyLong_Check(o)) return false;
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  *out = v;
  return true;
}

// softmax_scale argument: None is 1 / sqrt(D).
bool scale_of(PyObject* o, int64_t D, float* out) {
  if (o == Py_None) {
    *out = (float)(1.0 / std::sqrt((double)D));
    return true;
  }
  return number(o, out);
}

PyObject* none() { Py_RETURN_NONE; }

// Allocations and launches can block (a full queue, hipMalloc): other threads
// run meanwhile, as they do under ctypes and torch's own calls.
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// C++ exceptions (an allocation that fails, say) become Python ones, by torch's
// own translation.
template <class F>
PyObject* guarded(F f) {
  HANDLE_TH_ERRORS
  return f();
  END_HANDLE_TH_ERRORS
}

// dense_forward(q, k, v, scale, causal, left, right, with_lse, device, stream)
//   -> (out, lse or None) | status | None
PyObject* dense_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    int64_t left, right;
    fa_fwd_args p = {};
    if (n != 10 || !call_of(a[8], a[9], &c) || !integer(a[5], &left) || !integer(a[6], &right) ||
        !number(a[3], &p.softmax_scale))
      return none();
    const at::Tensor *q = plain(a[0], c, 4), *k = plain(a[1], c, 4), *v = plain(a[2], c, 4);
    if (!q || !k || !v || !half_code(*q, &p.dtype) || k->scalar_type() != q->scalar_type() ||
        v->scalar_type() != q->scalar_type() || !rows_ready(*q) || !rows_ready(*k) ||
        !rows_ready(*v))
      return none();
    const int64_t B = q->size(0), Sq = q->size(1), H = q->size(2), D = q->size(3);
    const int64_t Sk = k->size(1), Hk = k->size(2), lim = int64_t(1) << 24;
    if (k->sizes() != v->sizes() || k->size(0) != B || k->size(3) != D || H % Hk != 0 ||
        (D != 64 && D != 128 && D != 256) || k->stride(1) >= lim || v->stride(1) >= lim ||
        !fits(B) || !fits(Sq) || !fits(Sk) || !fits(H) || left < -1 || right < -1 || !fits(left) ||
        !fits(right))
      return none();
    const bool with_lse = a[7] == Py_True;
    const bool causal = a[4] == Py_True;
    at::Tensor out, lse;
    int status;
    {
      NoGil no_gil;
      out = at::empty({B, Sq, H, D}, q->options().requires_grad(false));
      if (with_lse) lse = at::empty({B, H, Sq}, out.options().dtype(at::kFloat));
      p.q = q->data_ptr();
      p.k = k->data_ptr();
      p.v = v->data_ptr();
      p.out = out.data_ptr();
      p.lse = with_lse ? lse.data_ptr<float>() : nullptr;
      set_strides(p.q_stride, *q);
      set_strides(p.k_stride, *k);
      set_strides(p.v_stride, *v);
      set_strides(p.o_stride, out);
      p.batch = (int32_t)B;
      p.seqlen_q = (int32_t)Sq;
      p.seqlen_k = (int32_t)Sk;
      p.num_heads = (int32_t)H;
      p.num_heads_k = (int32_t)Hk;
      p.head_dim = (int32_t)D;
      p.causal = causal;
      p.has_window = left != -1 || right != -1;
      p.window_left = (int32_t)left;
      p.window_right = (int32_t)right;
      status = lib.fwd(&p, c.stream);
    }
    if (status != FA_OK) return PyLong_FromLong(status);
    PyObject* l = with_lse ? THPVariable_Wrap(lse) : (Py_INCREF(Py_None), Py_None);
    return Py_BuildValue("NN", THPVariable_Wrap(out), l);
  });
}

// Caches [num_pages, page_size, kv_heads, head_dim] of q's dtype and head_dim,
// and the scalars every paged entry point shares.
template <class Args>
bool caches(const at::Tensor* q, const at::Tensor* kc, const at::Tensor* vc, PyObject* block_size,
            PyObject* num_kv_heads, PyObject* scale, Args* p) {
  int64_t page, heads;
  if (!q || !kc || !vc || !half_code(*q, &p->dtype) || kc->scalar_type() != q->scalar_type() ||
      vc->scalar_type() != q->scalar_type() || !rows_ready(*q) || !rows_ready(*kc) ||
      !rows_ready(*vc) || kc->sizes() != vc->sizes())
    return false;
  const int64_t H = q->size(1), D = q->size(2), Hk = kc->size(2), P = kc->size(1);
  if (!integer(block_size, &page) || page != P || (P & (P - 1)) != 0 || kc->size(3) != D ||
      (D != 64 && D != 128 && D != 256 && D != 512) || H % Hk != 0 || !fits(kc->size(0)) ||
      !fits(P) || !fits(H) || !scale_of(scale, D, &p->softmax_scale))
    return false;
  if (num_kv_heads != Py_None && !(integer(num_kv_heads, &heads) && (heads == 0 || heads == Hk)))
    return false;
  p->q = q->data_ptr();
  p->k_cache = kc->data_ptr();
  p->v_cache = vc->data_ptr();
  set_strides(p->q_stride, *q);
  set_strides(p->k_stride, *kc);
  set_strides(p->v_stride, *vc);
  p->num_heads = (int32_t)H;
  p->num_kv_heads = (int32_t)Hk;
  p->head_dim = (int32_t)D;
  p->page_size = (int32_t)P;
  p->num_pages = (int32_t)kc->size(0);
  return true;
}

template <class Args>
bool block_table(const at::Tensor* bt, const at::Tensor* seq_lens, int64_t batch, Args* p) {
  if (!index_ready(bt) || !index_ready(seq_lens) || bt->size(0) != batch ||
      seq_lens->size(0) != batch || !fits(batch) || !fits(bt->size(1) * p->page_size))
    return false;
  p->block_table = bt->data_ptr<int32_t>();
  p->seq_lens = seq_lens->data_ptr<int32_t>();
  p->block_table_stride = bt->size(1);
  p->max_blocks = (int32_t)bt->size(1);
  p->batch = (int32_t)batch;
  return true;
}

// decode(q, k_cache, v_cache, block_table, seq_lens, block_size, num_kv_heads, scale,
//        device, stream) -> out | status | None
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    fa_decode_args p = {};
    if (n != 10 || !call_of(a[8], a[9], &c)) return none();
    const at::Tensor* q = plain(a[0], c, 3);
    if (!caches(q, plain(a[1], c, 4), plain(a[2], c, 4), a[5], a[6], a[7], &p) ||
        !block_table(plain(a[3], c, 2), plain(a[4], c, 1), q->size(0), &p))
      return none();
    at::Tensor out;
    int status = FA_E_INVALID;
    {
      NoGil no_gil;
      out = at::empty(q->sizes(), q->options().requires_grad(false));
      p.out = out.data_ptr();
      set_strides(p.o_stride, out);
      p.max_seq_len = p.max_blocks * p.page_size;
      if (const size_t bytes = lib.decode_workspace(&p)) {
        at::Tensor ws = at::empty({(int64_t)bytes}, out.options().dtype(at::kByte));
        status = lib.decode(&p, ws.data_ptr(), bytes, c.stream);
      }
    }
    if (status != FA_OK) return PyLong_FromLong(status);
    return THPVariable_Wrap(out);
  });
}

// paged_forward(q, k_cache, v_cache, block_table, seq_lens, query_start_loc,
//               prefix_kv_lens, block_size, num_kv_heads, scale, causal, window_q, window_k,
//               device, stream) -> (out, lse) | status | None
PyObject* paged_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    fa_paged_args p = {};
    int64_t wq, wk;
    if (n != 15 || !call_of(a[13], a[14], &c) || !integer(a[11], &wq) || !integer(a[12], &wk) ||
        !fits(wq) || !fits(wk) || wq < INT_MIN || wk < INT_MIN)
      return none();
    const at::Tensor *q = plain(a[0], c, 3), *bt = plain(a[3], c, 2);
    if (!bt || !caches(q, plain(a[1], c, 4), plain(a[2], c, 4), a[7], a[8], a[9], &p) ||
        !block_table(bt, plain(a[4], c, 1), bt->size(0), &p) || !q->is_contiguous())
      return none();
    const at::Tensor *qsl = plain(a[5], c, 1), *prefix = plain(a[6], c, 1);
    if (!index_ready(qsl) || !index_ready(prefix) || qsl->size(0) != bt->size(0) + 1 ||
        prefix->size(0) != bt->size(0) || !fits(q->size(0)))
      return none();
    const bool causal = a[10] == Py_True;
    at::Tensor out, lse;
    int status;
    {
      NoGil no_gil;
      out = at::empty(q->sizes(), q->options().requires_grad(false));
      lse = at::empty({q->size(1), q->size(0)}, out.options().dtype(at::kFloat));
      p.out = out.data_ptr();
      p.lse = lse.data_ptr<float>();
      set_strides(p.o_stride, out);
      p.query_start_loc = qsl->data_ptr<int32_t>();
      p.prefix_kv_lens = prefix->data_ptr<int32_t>();
      p.num_tokens = (int32_t)q->size(0);
      p.causal = causal;
      p.window_q = (int32_t)wq;
      p.window_k = (int32_t)wk;
      status = lib.paged_splits(&p);
      if (status > 0) {
        const int splits = status;
        const size_t bytes = lib.paged_workspace(&p, splits);
        at::Tensor ws;
        if (bytes) ws = at::empty({(int64_t)bytes}, out.options().dtype(at::kByte));
        status = lib.paged(&p, splits, bytes ? ws.data_ptr() : nullptr, bytes, c.stream);
      }
    }
    if (status != FA_OK) return PyLong_FromLong(status);
    return Py_BuildValue("NN", THPVariable_Wrap(out), THPVariable_Wrap(lse));
  });
}

// cache_write(key, value, key_cache, value_cache, slot_mapping, device, stream)
//   -> 0 | status | None
PyObject* cache_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    fa_cache_write_args p = {};
    if (n != 7 || !call_of(a[5], a[6], &c)) return none();
    const at::Tensor *k = plain(a[0], c, 3), *v = plain(a[1], c, 3), *kc = plain(a[2], c, 4),
                     *vc = plain(a[3], c, 4), *slots = plain(a[4], c, 1);
    if (!k || !v || !kc || !vc || !slots || !half_code(*k, &p.dtype) ||
        v->scalar_type() != k->scalar_type() || kc->scalar_type() != k->scalar_type() ||
        vc->scalar_type() != k->scalar_type() || k->sizes() != v->sizes() ||
        kc->sizes() != vc->sizes() || kc->size(2) != k->size(1) || kc->size(3) != k->size(2) ||
        slots->scalar_type() != at::kLong || !slots->is_contiguous() ||
        slots->size(0) != k->size(0) || k->size(2) % 8 != 0 || k->size(2) > 1024 ||
        !rows_ready(*k) || !rows_ready(*v) || !rows_ready(*kc) || !rows_ready(*vc) ||
        !fits(k->size(0)) || !fits(k->size(1)) || !fits(kc->size(0)) || !fits(kc->size(1)))
      return none();
    p.key = k->data_ptr();
    p.value = v->data_ptr();
    p.k_cache = kc->data_ptr();
    p.v_cache = vc->data_ptr();
    p.slot_mapping = slots->data_ptr<int64_t>();
    set_strides(p.key_stride, *k);
    set_strides(p.value_stride, *v);
    set_strides(p.k_stride, *kc);
    set_strides(p.v_stride, *vc);
    p.num_tokens = (int32_t)k->size(0);
    p.num_kv_heads = (int32_t)k->size(1);
    p.head_dim = (int32_t)k->size(2);
    p.page_size = (int32_t)kc->size(1);
    p.num_pages = (int32_t)kc->size(0);
    int status;
    {
      NoGil no_gil;
      status = lib.cache_write(&p, c.stream);
    }
    return PyLong_FromLong(status);
  });
}

// ------------------------------------------------------------------ norm and rotation

bool same_half(const at::Tensor* t, const at::Tensor& like) {
  return t && t->scalar_type() == like.scalar_type() && rows_ready(*t);
}

// Position tables, weights (None: no norm), eps and the pairing, which the
// norm-and-rotation calls share.  `head` is a tensor [..., head_dim].
template <class Args>
bool rope_common(PyObject* cos_o, PyObject* sin_o, PyObject* qw_o, PyObject* kw_o, PyObject* eps,
                 PyObject* interleaved, const at::Tensor& head, const Call& c, Args* p) {
  const at::Tensor *cos = plain(cos_o, c, 2), *sin = plain(sin_o, c, 2);
  if (!cos || !sin || cos->scalar_type() != at::kFloat || sin->scalar_type() != at::kFloat ||
      cos->sizes() != sin->sizes() || cos->requires_grad() || sin->requires_grad())
    return false;
  const int64_t D = head.size(-1), R = 2 * cos->size(1);
  if (D % 8 != 0 || D < 16 || D > 512 || R % 16 != 0 || R < 16 || R > D) return false;
  const at::Tensor* tables[2] = {cos, sin};
  for (int i = 0; i < 2; ++i) {
    const at::Tensor& t = *tables[i];
    p->table_stride[i] = t.size(0) == 1 ? 0 : t.stride(0);
    if (t.stride(1) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0 ||
        p->table_stride[i] < 0 || p->table_stride[i] % 4 != 0)
      return false;
  }
  p->cos = cos->data_ptr<float>();
  p->sin = sin->data_ptr<float>();
  p->num_positions = cos->size(0);
  PyObject* weights[2] = {qw_o, kw_o};
  const void* ptr[2] = {nullptr, nullptr};
  int f32 = -1;
  for (int i = 0; i < 2; ++i) {
    if (weights[i] == Py_None) continue;
    const at::Tensor* w = plain(weights[i], c, 1);
    if (!w || w->size(0) != D || !w->is_contiguous() ||
        reinterpret_cast<uintptr_t>(w->data_ptr()) % 16 != 0)
      return false;
    const int is32 = w->scalar_type() == at::kFloat;
    if ((!is32 && w->scalar_type() != head.scalar_type()) || (f32 >= 0 && f32 != is32)) return false;
    f32 = is32;
    ptr[i] = w->data_ptr();
  }
  p->q_weight = ptr[0];
  p->k_weight = ptr[1];
  p->weight_f32 = f32 == 1;
  if (interleaved != Py_True && interleaved != Py_False) return false;
  p->interleaved = interleaved == Py_True;
  p->head_dim = (int32_t)D;
  p->rotary_dim = (int32_t)R;
  return number(eps, &p->eps);
}

// int64 [n], contiguous, or nullptr.
const int64_t* long_index(PyObject* o, const Call& c, int64_t n) {
  const at::Tensor* t = plain(o, c, 1);
  return t && t->scalar_type() == at::kLong && t->size(0) == n && t->is_contiguous()
             ? t->data_ptr<int64_t>()
             : nullptr;
}

// {batch, seq, head} strides of a [B, S, H, D] or [T, H, D] tensor.
void set_rows(int64_t (&dst)[3], const at::Tensor& t) {
  const int64_t n = t.dim() - 1;
  for (int64_t i = 0; i < n; ++i) dst[3 - n + i] = t.size(i) == 1 ? 0 : t.stride(i);
}

// Sizes and positions (None or a vector) of q / k, or of their gradients.
template <class Args>
bool rope_sizes(const at::Tensor& q, const at::Tensor& k, PyObject* positions, const Call& c,
                Args* p) {
  const int64_t d = q.dim();
  for (int64_t i = 0; i < d; ++i)
    if ((i != d - 2 && q.size(i) != k.size(i)) || !fits(q.size(i)) || !fits(k.size(i)))
      return false;
  if (positions != Py_None) {
    p->positions = long_index(positions, c, q.size(d - 3));
    if (!p->positions) return false;
    p->pos_stride[1] = 1;
  }
  p->batch = d == 4 ? (int32_t)q.size(0) : 1;
  p->seqlen = (int32_t)q.size(d - 3);
  p->num_heads = (int32_t)q.size(d - 2);
  p->num_heads_k = (int32_t)k.size(d - 2);
  return true;
}

// A plain tensor [B, S, H, D] or [T, H, D].
const at::Tensor* plain_heads(PyObject* o, const Call& c) {
  const at::Tensor* t = plain(o, c, 4);
  return t ? t : plain(o, c, 3);
}

// fa_norm_rope on checked tensors (p holds what rope_common and rope_sizes set).
int rope_forward(fa_norm_rope_args p, const at::Tensor& q, const at::Tensor& k, void* stream,
                 at::Tensor* q_out, at::Tensor* k_out) {
  *q_out = at::empty(q.sizes(), q.options().requires_grad(false));
  *k_out = at::empty(k.sizes(), q_out->options());
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.q_out = q_out->data_ptr();
  p.k_out = k_out->data_ptr();
  set_rows(p.q_stride, q);
  set_rows(p.k_stride, k);
  set_rows(p.qo_stride, *q_out);
  set_rows(p.ko_stride, *k_out);
  return lib.norm_rope(&p, stream);
}

struct RopeGrads {
  at::Tensor dq, dk, dqw, dkw;
};
// fa_norm_rope_bwd: gq, gk the outputs' gradients, q and k (read where their weight is).
int rope_backward(fa_norm_rope_bwd_args p, const at::Tensor& q, const at::Tensor& k,
                  const at::Tensor& gq, const at::Tensor& gk, void* stream, RopeGrads* r) {
  r->dq = at::empty(gq.sizes(), gq.options().requires_grad(false));
  r->dk = at::empty(gk.sizes(), r->dq.options());
  const auto w = r->dq.options().dtype(p.weight_f32 ? at::kFloat : gq.scalar_type());
  if (p.q_weight) {
    r->dqw = at::empty({p.head_dim}, w);
    p.q = q.data_ptr();
    set_rows(p.q_stride, q);
    p.dq_weight = r->dqw.data_ptr();
  }
  if (p.k_weight) {
    r->dkw = at::empty({p.head_dim}, w);
    p.k = k.data_ptr();
    set_rows(p.k_stride, k);
    p.dk_weight = r->dkw.data_ptr();
  }
  p.dq_out = gq.data_ptr();
  p.dk_out = gk.data_ptr();
  p.dq = r->dq.data_ptr();
  p.dk = r->dk.data_ptr();
  set_rows(p.dqo_stride, gq);
  set_rows(p.dko_stride, gk);
  set_rows(p.dq_stride, r->dq);
  set_rows(p.dk_stride, r->dk);
  const size_t bytes = lib.norm_rope_bwd_workspace(&p);
  at::Tensor ws;
  if (bytes) ws = at::empty({(int64_t)bytes}, r->dq.options().dtype(at::kByte));
  return lib.norm_rope_bwd(&p, bytes ? ws.data_ptr() : nullptr, bytes, stream);
}

// What a node of this file shares: the stream its forward ran on, which is the one
// the engine makes current for its backward.
struct FaNode : torch::autograd::Node {
  void* stream = nullptr;
  std::mutex lock;

  // An output's gradient as the kernels take it: zeros where there is none.
  static at::Tensor ready(const at::Tensor& g, at::IntArrayRef size, const at::TensorOptions& o) {
    if (!g.defined()) return at::zeros(size, o);
    at::Tensor t = g.scalar_type() == o.dtype().toScalarType() ? g : g.to(o.dtype());
    return rows_ready(t) ? t : t.clone(at::MemoryFormat::Contiguous);
  }
  // The gradients, which themselves have none: differentiating them is an error.
  static torch::autograd::variable_list once(torch::autograd::variable_list&& out,
                                             const torch::autograd::variable_list& grads) {
    bool again = false;
    for (const auto& g : grads) again |= g.defined() && g.requires_grad();
    if (!again || !at::GradMode::is_enabled()) return std::move(out);
    auto stop = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that can be differentiated once",
        (int64_t)out.size());
    for (auto& t : out)
      if (t.defined()) t = t.detach().set_requires_grad(true);
    return (*stop)(std::move(out));
  }
};

struct RopeNode : FaNode {
  torch::autograd::SavedVariable q, k, cos, sin, qw, kw, pos;
  bool has_q = false, has_k = false, has_pos = false;
  std::vector<int64_t> q_size, k_size;
  at::TensorOptions options;
  fa_norm_rope_args p = {};

  std::string name() const override { return "QkNormRopeBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> hold(lock);
    for (auto* v : {&q, &k, &cos, &sin, &qw, &kw, &pos}) v->reset_data();
  }
  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    std::lock_guard<std::mutex> hold(lock);
    at::Tensor c = cos.unpack(), s = sin.unpack(), x, y, a, b, t;
    if (has_q) x = q.unpack(), a = qw.unpack();
    if (has_k) y = k.unpack(), b = kw.unpack();
    if (has_pos) t = pos.unpack();
    RopeGrads r;
    {
      at::NoGradGuard none;
      const at::Tensor gq = ready(grads[0], q_size, options), gk = ready(grads[1], k_size, options);
      fa_norm_rope_bwd_args n = {};
      n.q_weight = has_q ? a.data_ptr() : nullptr;
      n.k_weight = has_k ? b.data_ptr() : nullptr;
      n.cos = c.data_ptr<float>();
      n.sin = s.data_ptr<float>();
      n.positions = has_pos ? t.data_ptr<int64_t>() : nullptr;
      for (int i = 0; i < 2; ++i) {
        n.table_stride[i] = p.table_stride[i];
        n.pos_stride[i] = p.pos_stride[i];
      }
      n.num_positions = p.num_positions;
      n.batch = p.batch;
      n.seqlen = p.seqlen;
      n.num_heads = p.num_heads;
      n.num_heads_k = p.num_heads_k;
      n.head_dim = p.head_dim;
      n.rotary_dim = p.rotary_dim;
      n.interleaved = p.interleaved;
      n.weight_f32 = p.weight_f32;
      n.dtype = p.dtype;
      n.eps = p.eps;
      const int status = rope_backward(n, x, y, gq, gk, stream, &r);
      TORCH_CHECK(status == FA_OK, "fa_norm_rope_bwd: status ", status);
    }
    return once({r.dq, r.dk, r.dqw, r.dkw}, grads);
  }
};

at::Tensor or_undefined(PyObject* o) {
  return o == Py_None ? at::Tensor() : THPVariable_Unpack(o);
}

// norm_rope(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved, with_grad,
//           device, stream) -> (q_out, k_out) | status | None.  Positions: None or a vector.
// with_grad True: the outputs have a node in the autograd graph; None: a call that
// would need one is handed back.
PyObject* norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    fa_norm_rope_args p = {};
    if (n != 12 || !call_of(a[10], a[11], &c)) return none();
    const at::Tensor *q = plain_heads(a[0], c), *k = plain_heads(a[1], c);
    if (!q || !k || q->dim() != k->dim() || !half_code(*q, &p.dtype) || !rows_ready(*q) ||
        !same_half(k, *q) || !rope_common(a[2], a[3], a[4], a[5], a[7], a[8], *q, c, &p) ||
        !rope_sizes(*q, *k, a[6], c, &p))
      return none();
    const bool with_grad = a[9] == Py_True;
    if (a[9] == Py_None && at::GradMode::is_enabled())
      for (int i : {0, 1, 4, 5})
        if (a[i] != Py_None && THPVariable_Unpack(a[i]).requires_grad()) return none();
    const at::Tensor cos = or_undefined(a[2]), sin = or_undefined(a[3]), qw = or_undefined(a[4]),
                     kw = or_undefined(a[5]), pos = or_undefined(a[6]);
    at::Tensor q_out, k_out;
    int status;
    {
      NoGil no_gil;
      status = rope_forward(p, *q, *k, c.stream, &q_out, &k_out);
      if (status == FA_OK && with_grad) {
        auto node = std::shared_ptr<RopeNode>(new RopeNode(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(*q, *k, qw, kw));
        node->stream = c.stream;
        node->p = p;
        node->q_size = q->sizes().vec();
        node->k_size = k->sizes().vec();
        node->options = q_out.options();
        using torch::autograd::SavedVariable;
        if ((node->has_q = qw.defined())) {
          node->q = SavedVariable(*q, false);
          node->qw = SavedVariable(qw, false);
        }
        if ((node->has_k = kw.defined())) {
          node->k = SavedVariable(*k, false);
          node->kw = SavedVariable(kw, false);
        }
        if ((node->has_pos = pos.defined())) node->pos = SavedVariable(pos, false);
        node->cos = SavedVariable(cos, false);
        node->sin = SavedVariable(sin, false);
        torch::autograd::set_history(q_out, node);
        torch::autograd::set_history(k_out, node);
      }
    }
    if (status != FA_OK) return PyLong_FromLong(status);
    return Py_BuildValue("NN", THPVariable_Wrap(q_out), THPVariable_Wrap(k_out));
  });
}

// norm_rope_bwd(q, k, dq_out, dk_out, cos, sin, q_weight, k_weight, positions, eps, interleaved,
//               device, stream) -> (dq, dk, dq_weight, dk_weight) | status | None.
// q / k and the weights' gradients are None where the weight is.
PyObject* norm_rope_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    fa_norm_rope_bwd_args p = {};
    if (n != 13 || !call_of(a[11], a[12], &c)) return none();
    const at::Tensor *gq = plain_heads(a[2], c), *gk = plain_heads(a[3], c);
    if (!gq || !gk || gq->dim() != gk->dim() || !half_code(*gq, &p.dtype) || !rows_ready(*gq) ||
        !same_half(gk, *gq) || !rope_common(a[4], a[5], a[6], a[7], a[9], a[10], *gq, c, &p) ||
        !rope_sizes(*gq, *gk, a[8], c, &p))
      return none();
    at::Tensor q, k;
    if (p.q_weight) {
      const at::Tensor* t = plain_heads(a[0], c);
      if (!same_half(t, *gq) || t->sizes() != gq->sizes()) return none();
      q = *t;
    }
    if (p.k_weight) {
      const at::Tensor* t = plain_heads(a[1], c);
      if (!same_half(t, *gq) || t->sizes() != gk->sizes()) return none();
      k = *t;
    }
    RopeGrads r;
    int status;
    {
      NoGil no_gil;
      status = rope_backward(p, q, k, *gq, *gk, c.stream, &r);
    }
    if (status != FA_OK) return PyLong_FromLong(status);
    auto or_none = [](const at::Tensor& t) {
      return t.defined() ? THPVariable_Wrap(t) : (Py_INCREF(Py_None), Py_None);
    };
    return Py_BuildValue("NNNN", THPVariable_Wrap(r.dq), THPVariable_Wrap(r.dk), or_none(r.dqw),
                         or_none(r.dkw));
  });
}

// norm_rope_cache(q, k, v, key_cache, value_cache, slot_mapping, positions, cos, sin,
//                 q_weight, k_weight, eps, interleaved, device, stream) -> q_out | status | None
PyObject* norm_rope_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    fa_norm_rope_cache_args p = {};
    if (n != 15 || !call_of(a[13], a[14], &c)) return none();
    const at::Tensor *q = plain(a[0], c, 3), *k = plain(a[1], c, 3), *v = plain(a[2], c, 3),
                     *kc = plain(a[3], c, 4), *vc = plain(a[4], c, 4);
    if (!q || !half_code(*q, &p.dtype) || !rows_ready(*q) || !same_half(k, *q) ||
        !same_half(v, *q) || !same_half(kc, *q) || !same_half(vc, *q) ||
        k->sizes() != v->sizes() || kc->sizes() != vc->sizes() || kc->size(2) != k->size(1) ||
        kc->size(3) != k->size(2) || q->size(0) != k->size(0) || q->size(2) != k->size(2) ||
        !fits(q->size(0)) || !fits(q->size(1)) || !fits(k->size(1)) || !fits(kc->size(0)) ||
        !fits(kc->size(1)) ||
        !rope_common(a[7], a[8], a[9], a[10], a[11], a[12], *q, c, &p))
      return none();
    p.slot_mapping = long_index(a[5], c, q->size(0));
    p.positions = long_index(a[6], c, q->size(0));
    if (!p.slot_mapping || !p.positions) return none();
    at::Tensor out;
    int status;
    {
      NoGil no_gil;
      out = at::empty(q->sizes(), q->options().requires_grad(false));
      p.q = q->data_ptr();
      p.k = k->data_ptr();
      p.v = v->data_ptr();
      p.q_out = out.data_ptr();
      p.k_cache = kc->data_ptr();
      p.v_cache = vc->data_ptr();
      set_strides(p.q_stride, *q);
      set_strides(p.key_stride, *k);
      set_strides(p.value_stride, *v);
      set_strides(p.qo_stride, out);
      set_strides(p.k_stride, *kc);
      set_strides(p.v_stride, *vc);
      p.num_tokens = (int32_t)q->size(0);
      p.num_heads = (int32_t)q->size(1);
      p.num_kv_heads = (int32_t)k->size(1);
      p.num_pages = (int32_t)kc->size(0);
      p.page_size = (int32_t)kc->size(1);
      status = lib.norm_rope_cache(&p, c.stream);
    }
    if (status != FA_OK) return PyLong_FromLong(status);
    return THPVariable_Wrap(out);
  });
}

// ------------------------------------------------------------------ linear attention

// q [n, H, D], k, v [n, Hk, D], log_decay [H], a state pool [N, H, D, D], slots
// (None or int32 [batch]) and the scale, of the serving calls.  `batch`: sequences.
template <class Args>
bool linear_common(PyObject* const* a, PyObject* slots_o, PyObject* scale, int64_t batch,
                   const Call& c, const at::Tensor* q, Args* p, const at::Tensor** state) {
  const at::Tensor *k = plain(a[1], c, 3), *v = plain(a[2], c, 3), *g = plain(a[3], c, 1),
                   *s = plain(a[4], c, 4);
  if (!half_code(*q, &p->dtype) || !rows_ready(*q) || !same_half(k, *q) || !same_half(v, *q) ||
      k->sizes() != v->sizes() || k->size(0) != q->size(0) || k->size(2) != q->size(2) || !g || !s)
    return false;
  const int64_t H = q->size(1), Hk = k->size(1), D = q->size(2);
  if ((D != 64 && D != 128 && D != 256) || H % Hk != 0 || !fits(H) || !fits(q->size(0)) ||
      g->scalar_type() != at::kFloat || g->size(0) != H || !g->is_contiguous() ||
      g->requires_grad() || s->scalar_type() != at::kFloat || s->size(1) != H ||
      s->size(2) != D || s->size(3) != D || !fits(s->size(0)) || !s->is_contiguous() ||
      reinterpret_cast<uintptr_t>(s->data_ptr()) % 16 != 0 || !scale_of(scale, D, &p->scale))
    return false;
  if (slots_o != Py_None) {
    const at::Tensor* slots = plain(slots_o, c, 1);
    if (!index_ready(slots) || slots->size(0) != batch) return false;
    p->state_indices = slots->data_ptr<int32_t>();
  } else if (batch > s->size(0)) {
    return false;
  }
  p->q = q->data_ptr();
  p->k = k->data_ptr();
  p->v = v->data_ptr();
  p->log_decay = g->data_ptr<float>();
  p->num_heads = (int32_t)H;
  p->num_heads_k = (int32_t)Hk;
  p->head_dim = (int32_t)D;
  p->num_states = (int32_t)s->size(0);
  p->batch = (int32_t)batch;
  *state = s;
  return true;
}

// Dense q [B, S, H, D], k, v [B, S, Hk, D] and log_decay [H].
template <class Args>
bool linear_dense(const at::Tensor* q, const at::Tensor* k, const at::Tensor* v, PyObject* decay,
                  PyObject* scale, const Call& c, Args* p) {
  const at::Tensor* g = plain(decay, c, 1);
  if (!q || !half_code(*q, &p->dtype) || !rows_ready(*q) || !same_half(k, *q) ||
      !same_half(v, *q) || k->sizes() != v->sizes() || k->size(0) != q->size(0) ||
      k->size(1) != q->size(1) || k->size(3) != q->size(3) || !g || !number(scale, &p->scale))
    return false;
  const int64_t H = q->size(2), Hk = k->size(2), D = q->size(3), lim = int64_t(1) << 24;
  if ((D != 64 && D != 128 && D != 256) || H % Hk != 0 || !fits(H) || !fits(q->size(0)) ||
      !fits(q->size(1)) || q->stride(1) >= lim || k->stride(1) >= lim || v->stride(1) >= lim ||
      g->scalar_type() != at::kFloat || g->size(0) != H || !g->is_contiguous() ||
      g->requires_grad())
    return false;
  p->q = q->data_ptr();
  p->k = k->data_ptr();
  p->v = v->data_ptr();
  p->log_decay = g->data_ptr<float>();
  set_strides(p->q_stride, *q);
  set_strides(p->k_stride, *k);
  set_strides(p->v_stride, *v);
  p->batch = (int32_t)q->size(0);
  p->seqlen = (int32_t)q->size(1);
  p->num_heads = (int32_t)H;
  p->num_heads_k = (int32_t)Hk;
  p->head_dim = (int32_t)D;
  return true;
}

// None, or a contiguous fp32 [B, H, D, D] state of q's sizes: its data and strides.
template <size_t N>
bool state_of(PyObject* o, const at::Tensor& q, const Call& c, const float** data,
              int64_t (&stride)[N]) {
  if (o == Py_None) return true;
  const at::Tensor* s = plain(o, c, 4);
  if (!s || s->scalar_type() != at::kFloat || s->size(0) != q.size(0) ||
      s->size(1) != q.size(2) || s->size(2) != q.size(3) || s->size(3) != q.size(3) ||
      !s->is_contiguous() || reinterpret_cast<uintptr_t>(s->data_ptr()) % 16 != 0)
    return false;
  *data = s->data_ptr<float>();
  set_strides(stride, *s);
  return true;
}

struct LinearGrads {
  at::Tensor dq, dk, dv, ds;
};
// fa_linear_bwd on checked tensors (p holds what linear_dense and state_of set).
int linear_backward(fa_linear_bwd_args p, const at::Tensor& q, const at::Tensor& k,
                    const at::Tensor& g, bool want_state, void* stream, LinearGrads* r) {
  r->dq = at::empty(q.sizes(), q.options().requires_grad(false));
  r->dk = at::empty(k.sizes(), r->dq.options());
  r->dv = at::empty(k.sizes(), r->dq.options());
  p.dout = g.data_ptr();
  p.dq = r->dq.data_ptr();
  p.dk = r->dk.data_ptr();
  p.dv = r->dv.data_ptr();
  set_strides(p.do_stride, g);
  set_strides(p.dq_stride, r->dq);
  set_strides(p.dk_stride, r->dk);
  set_strides(p.dv_stride, r->dv);
  if (want_state) {
    r->ds = at::empty({q.size(0), q.size(2), q.size(3), q.size(3)},
                      r->dq.options().dtype(at::kFloat));
    p.d_initial_state = r->ds.data_ptr<float>();
    set_strides(p.dis_stride, r->ds);
  }
  const size_t bytes = lib.linear_bwd_workspace(&p);
  at::Tensor ws;
  if (bytes) ws = at::empty({(int64_t)bytes}, r->dq.options().dtype(at::kByte));
  return lib.linear_bwd(&p, bytes ? ws.data_ptr() : nullptr, bytes, stream);
}

struct LinearNode : FaNode {
  torch::autograd::SavedVariable q, k, v, decay, init;
  bool has_init = false, want_init = false;
  std::vector<int64_t> state_size;
  fa_linear_args p = {};

  std::string name() const override { return "LinearAttnBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> hold(lock);
    for (auto* x : {&q, &k, &v, &decay, &init}) x->reset_data();
  }
  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    std::lock_guard<std::mutex> hold(lock);
    const at::Tensor tq = q.unpack(), tk = k.unpack(), tv = v.unpack(), td = decay.unpack();
    at::Tensor ti;
    if (has_init) ti = init.unpack();
    LinearGrads r;
    {
      at::NoGradGuard none;
      at::Tensor g = ready(grads[0], tq.sizes(), tq.options().requires_grad(false));
      if (g.stride(1) >= (int64_t(1) << 24)) g = g.clone(at::MemoryFormat::Contiguous);
      at::Tensor ds;
      if (grads.size() > 1 && grads[1].defined()) {
        ds = grads[1].to(at::kFloat).contiguous();
        if (reinterpret_cast<uintptr_t>(ds.data_ptr()) % 16 != 0)
          ds = ds.clone(at::MemoryFormat::Contiguous);
      }
      fa_linear_bwd_args n = {};
      n.q = tq.data_ptr();
      n.k = tk.data_ptr();
      n.v = tv.data_ptr();
      n.log_decay = td.data_ptr<float>();
      for (int i = 0; i < 3; ++i) {
        n.q_stride[i] = p.q_stride[i];
        n.k_stride[i] = p.k_stride[i];
        n.v_stride[i] = p.v_stride[i];
      }
      if (has_init) {
        n.initial_state = ti.data_ptr<float>();
        set_strides(n.is_stride, ti);
      }
      if (ds.defined()) {
        n.d_final_state = ds.data_ptr<float>();
        set_strides(n.fs_stride, ds);
      }
      n.batch = p.batch;
      n.seqlen = p.seqlen;
      n.num_heads = p.num_heads;
      n.num_heads_k = p.num_heads_k;
      n.head_dim = p.head_dim;
      n.scale = p.scale;
      n.dtype = p.dtype;
      const int status = linear_backward(n, tq, tk, g, want_init, stream, &r);
      TORCH_CHECK(status == FA_OK, "fa_linear_bwd: status ", status);
    }
    return once({r.dq, r.dk, r.dv, r.ds}, grads);
  }
};

// linear_dense_fwd(q, k, v, log_decay, scale, initial_state, want_final, with_grad, device,
//                  stream) -> (out, final_state or None) | status | None
PyObject* linear_dense_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    fa_linear_args p = {};
    if (n != 10 || !call_of(a[8], a[9], &c)) return none();
    const at::Tensor *q = plain(a[0], c, 4), *k = plain(a[1], c, 4), *v = plain(a[2], c, 4);
    if (!linear_dense(q, k, v, a[3], a[4], c, &p) ||
        !state_of(a[5], *q, c, &p.initial_state, p.is_stride))
      return none();
    const bool want_final = a[6] == Py_True, with_grad = a[7] == Py_True;
    const at::Tensor decay = or_undefined(a[3]), init = or_undefined(a[5]);
    at::Tensor out, fin;
    int status;
    {
      NoGil no_gil;
      out = at::empty(q->sizes(), q->options().requires_grad(false));
      p.out = out.data_ptr();
      set_strides(p.o_stride, out);
      p.num_states = p.batch;
      if (want_final) {
        fin = at::empty({q->size(0), q->size(2), q->size(3), q->size(3)},
                        out.options().dtype(at::kFloat));
        p.final_state = fin.data_ptr<float>();
        set_strides(p.fs_stride, fin);
      }
      const size_t bytes = lib.linear_workspace(&p);
      at::Tensor ws;
      if (bytes) ws = at::empty({(int64_t)bytes}, out.options().dtype(at::kByte));
      status = lib.linear_fwd(&p, bytes ? ws.data_ptr() : nullptr, bytes, c.stream);
      if (status == FA_OK && with_grad) {
        auto node = std::shared_ptr<LinearNode>(new LinearNode(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(*q, *k, *v, init));
        node->stream = c.stream;
        node->p = p;
        using torch::autograd::SavedVariable;
        node->q = SavedVariable(*q, false);
        node->k = SavedVariable(*k, false);
        node->v = SavedVariable(*v, false);
        node->decay = SavedVariable(decay, false);
        if ((node->has_init = init.defined())) {
          node->init = SavedVariable(init, false);
          node->want_init = init.requires_grad();
        }
        torch::autograd::set_history(out, node);
        if (want_final) torch::autograd::set_history(fin, node);
      }
    }
    if (status != FA_OK) return PyLong_FromLong(status);
    PyObject* f = want_final ? THPVariable_Wrap(fin) : (Py_INCREF(Py_None), Py_None);
    return Py_BuildValue("NN", THPVariable_Wrap(out), f);
  });
}

// linear_dense_bwd(q, k, v, dout, log_decay, scale, initial_state, d_final_state,
//                  want_d_initial, device, stream)
//   -> (dq, dk, dv, d_initial_state or None) | status | None
PyObject* linear_dense_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    fa_linear_bwd_args p = {};
    if (n != 11 || !call_of(a[9], a[10], &c)) return none();
    const at::Tensor *q = plain(a[0], c, 4), *k = plain(a[1], c, 4), *v = plain(a[2], c, 4),
                     *g = plain(a[3], c, 4);
    if (!linear_dense(q, k, v, a[4], a[5], c, &p) || !same_half(g, *q) ||
        g->sizes() != q->sizes() || g->stride(1) >= (int64_t(1) << 24) ||
        !state_of(a[6], *q, c, &p.initial_state, p.is_stride) ||
        !state_of(a[7], *q, c, &p.d_final_state, p.fs_stride))
      return none();
    const bool want = a[8] == Py_True;
    LinearGrads r;
    int status;
    {
      NoGil no_gil;
      status = linear_backward(p, *q, *k, *g, want, c.stream, &r);
    }
    if (status != FA_OK) return PyLong_FromLong(status);
    PyObject* d = want ? THPVariable_Wrap(r.ds) : (Py_INCREF(Py_None), Py_None);
    return Py_BuildValue("NNNN", THPVariable_Wrap(r.dq), THPVariable_Wrap(r.dk),
                         THPVariable_Wrap(r.dv), d);
  });
}

// linear_prefill(q, k, v, log_decay, state, query_start_loc, prefix_kv_lens, state_indices,
//                scale, device, stream) -> out | status | None
PyObject* linear_prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    fa_linear_args p = {};
    if (n != 11 || !call_of(a[9], a[10], &c)) return none();
    const at::Tensor *q = plain(a[0], c, 3), *starts = plain(a[5], c, 1),
                     *prefix = plain(a[6], c, 1), *state = nullptr;
    if (!q || !index_ready(starts) || !index_ready(prefix) ||
        starts->size(0) != prefix->size(0) + 1 || !fits(prefix->size(0)) ||
        !linear_common(a, a[7], a[8], prefix->size(0), c, q, &p, &state))
      return none();
    const at::Tensor &k = THPVariable_Unpack(a[1]), &v = THPVariable_Unpack(a[2]);
    const int64_t lim = int64_t(1) << 24;
    if (q->stride(0) >= lim || k.stride(0) >= lim || v.stride(0) >= lim) return none();
    at::Tensor out;
    int status;
    {
      NoGil no_gil;
      out = at::empty(q->sizes(), q->options().requires_grad(false));
      auto put = [](int64_t (&dst)[3], const at::Tensor& t) {
        dst[1] = t.size(0) == 1 ? 0 : t.stride(0);
        dst[2] = t.size(1) == 1 ? 0 : t.stride(1);
      };
      put(p.q_stride, *q);
      put(p.k_stride, k);
      put(p.v_stride, v);
      put(p.o_stride, out);
      p.out = out.data_ptr();
      p.initial_state = p.final_state = state->data_ptr<float>();
      set_strides(p.is_stride, *state);
      set_strides(p.fs_stride, *state);
      p.query_start_loc = starts->data_ptr<int32_t>();
      p.prefix_kv_lens = prefix->data_ptr<int32_t>();
      p.seqlen = (int32_t)q->size(0);
      const size_t bytes = lib.linear_workspace(&p);
      at::Tensor ws;
      if (bytes) ws = at::empty({(int64_t)bytes}, out.options().dtype(at::kByte));
      status = lib.linear_fwd(&p, bytes ? ws.data_ptr() : nullptr, bytes, c.stream);
    }
    if (status != FA_OK) return PyLong_FromLong(status);
    return THPVariable_Wrap(out);
  });
}

// linear_decode(q, k, v, log_decay, state, state_indices, scale, device, stream)
//   -> out | status | None
PyObject* linear_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    fa_linear_decode_args p = {};
    if (n != 9 || !call_of(a[7], a[8], &c)) return none();
    const at::Tensor *q = plain(a[0], c, 3), *state = nullptr;
    if (!q || !linear_common(a, a[5], a[6], q->size(0), c, q, &p, &state)) return none();
    at::Tensor out;
    int status;
    {
      NoGil no_gil;
      out = at::empty(q->sizes(), q->options().requires_grad(false));
      set_strides(p.q_stride, *q);
      set_strides(p.k_stride, THPVariable_Unpack(a[1]));
      set_strides(p.v_stride, THPVariable_Unpack(a[2]));
      set_strides(p.o_stride, out);
      set_strides(p.s_stride, *state);
      p.out = out.data_ptr();
      p.state = state->data_ptr<float>();
      status = lib.linear_decode(&p, c.stream);
    }
    if (status != FA_OK) return PyLong_FromLong(status);
    return THPVariable_Wrap(out);
  });
}

// foreign_leaf(tensor) -> bool: a leaf whose gradient accumulator a graph made on
// another stream keeps alive.  The engine records an event on that stream when the
// backward ends, which a stream capture does not survive (the process ends).
PyObject* foreign_leaf(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 1 || !THPVariable_Check(a[0])) Py_RETURN_FALSE;
    const at::Tensor& t = THPVariable_Unpack(a[0]);
    if (!t.defined() || !t.is_cuda() || !t.requires_grad() || !t.is_leaf()) Py_RETURN_FALSE;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node || !node->stream()) Py_RETURN_FALSE;
    const c10::impl::VirtualGuardImpl guard(c10::DeviceType::CUDA);
    if (*node->stream() != guard.getStream(t.device())) Py_RETURN_TRUE;
    Py_RETURN_FALSE;
  });
}

// bind(...): the library's entry points, as addresses, in the order of Entries.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr int kEntries = 16;
  void* f[kEntries];
  if (n != kEntries) {
    PyErr_Format(PyExc_TypeError, "bind takes %d addresses", kEntries);
    return nullptr;
  }
  for (int i = 0; i < kEntries; ++i) {
    f[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  lib = {reinterpret_cast<decltype(lib.fwd)>(f[0]),
         reinterpret_cast<decltype(lib.decode_workspace)>(f[1]),
         reinterpret_cast<decltype(lib.decode)>(f[2]),
         reinterpret_cast<decltype(lib.paged_splits)>(f[3]),
         reinterpret_cast<decltype(lib.paged_workspace)>(f[4]),
         reinterpret_cast<decltype(lib.paged)>(f[5]),
         reinterpret_cast<decltype(lib.cache_write)>(f[6]),
         reinterpret_cast<decltype(lib.norm_rope)>(f[7]),
         reinterpret_cast<decltype(lib.norm_rope_cache)>(f[8]),
         reinterpret_cast<decltype(lib.linear_workspace)>(f[9]),
         reinterpret_cast<decltype(lib.linear_fwd)>(f[10]),
         reinterpret_cast<decltype(lib.linear_decode)>(f[11]),
         reinterpret_cast<decltype(lib.norm_rope_bwd_workspace)>(f[12]),
         reinterpret_cast<decltype(lib.norm_rope_bwd)>(f[13]),
         reinterpret_cast<decltype(lib.linear_bwd_workspace)>(f[14]),
         reinterpret_cast<decltype(lib.linear_bwd)>(f[15])};
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL,
          nullptr};
}

PyMethodDef methods[] = {method<bind>("bind"),
                         method<dense_forward>("dense_forward"),
                         method<decode>("decode"),
                         method<paged_forward>("paged_forward"),
                         method<cache_write>("cache_write"),
                         method<norm_rope>("norm_rope"),
                         method<norm_rope_cache>("norm_rope_cache"),
                         method<norm_rope_bwd>("norm_rope_bwd"),
                         method<linear_dense_fwd>("linear_dense_fwd"),
                         method<linear_dense_bwd>("linear_dense_bwd"),
                         method<linear_prefill>("linear_prefill"),
                         method<linear_decode>("linear_decode"),
                         method<foreign_leaf>("foreign_leaf"),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_fa_torch", nullptr, -1, methods};

}  // namespace

// FA_TORCH_VERSION: the torch whose headers this was compiled against; another
// one's tensors may be laid out differently, so the loader compares it.
PyMODINIT_FUNC PyInit__fa_torch(void) {
  PyObject* m = PyModule_Create(&module_def);
  if (m && PyModule_AddStringConstant(m, "torch_version", FA_TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
