// The common case of the eager calls of the decoder operators (quantize_rows, gemm_rcr_int8, rotary_embedding,
// paged_kv_append, prefix_attention, gemm_rcr_lora, qk_norm_rotary, token_logprobs), without the interpreter: see native_calls.cpp, whose rules these follow.  One token's
// rotation takes 3 us on the GPU and took 16 through Python's attribute reads, checks and ctypes.
//
// Beside what native_calls.cpp asks for, every tensor has to be on the current device: the Python path changes it where it is
// another.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/PyInterpreter.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/headeronly/version.h>

#include <ATen/Context.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPFunctions.h>

#include <cmath>

#include "../../include/aitemplate_amd_kernels.h"
#include "native_device.h"

#ifndef AITAMD_TORCH_BUILD
#define AITAMD_TORCH_BUILD TORCH_VERSION
#endif

namespace {

#include "native_common.inc"

// Tensors read so far that are all ordinary: of a type each, on the current device
struct Operands {
  bool ok = true;
  int device = -1;  // (asked for behind the first tensor on one: there may be none)
  bool here(const at::Tensor& t) {
    if (device < 0) device = c10::hip::current_device();
    return t.device().index() == device;
  }
  const at::Tensor* get(PyObject* o, at::ScalarType type) {
    const at::Tensor* t = gpu_tensor(o);
    if (t == nullptr || t->scalar_type() != type || !here(*t)) {
      ok = false;
      return nullptr;
    }
    return t;
  }
  const at::Tensor* optional(PyObject* o, at::ScalarType type) { return o == Py_None ? nullptr : get(o, type); }
};

bool dense(const at::Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }

bool number(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

at::Tensor make(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

// the first tensor of a call, which gives the type of the others; its type id or -1
int first_operand(PyObject* o, Operands& ops, const at::Tensor** t) {
  *t = gpu_tensor(o);
  const int dt = *t == nullptr ? -1 : dtype_id(**t);
  return dt >= 0 && ops.here(**t) ? dt : -1;
}

PyObject* pair_of(int rc, const char* what, const at::Tensor& a, const at::Tensor& b) {
  if (rc != 0) return PyErr_Format(PyExc_RuntimeError, "%s failed: %s", what, aitamd_last_error());
  THPObjectPtr x(THPVariable_Wrap(a)), y(THPVariable_Wrap(b));
  return x && y ? PyTuple_Pack(2, x.get(), y.get()) : nullptr;
}

// quantize_rows(x): new results only
PyObject* quantize_rows(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    if (nargs != 1 || !plain_allocation()) return not_ordinary();
    Operands ops;
    const at::Tensor* x;
    const int dt = first_operand(args[0], ops, &x);
    if (dt < 0 || x->dim() < 1 || x->numel() == 0) return not_ordinary();
    const int64_t columns = x->size(-1), rows = x->numel() / columns;
    int64_t ldx;
    if (!flat_row_pitch(*x, rows, columns, &ldx)) return not_ordinary();
    at::Tensor q = make(x->sizes(), at::kChar, *x), scale = make(x->sizes().slice(0, x->dim() - 1), at::kFloat, *x);
    const void* px = x->data_ptr();
    int8_t* pq = static_cast<int8_t*>(q.data_ptr());
    float* ps = static_cast<float*>(scale.data_ptr());
    void* stream = current_stream();
    const int rc = unlocked([&] { return aitamd_quantize_rows(dt, px, pq, ps, rows, columns, ldx, columns, stream); });
    return pair_of(rc, "quantize_rows", q, scale);
  });
}

// whether rows of K bytes, `pitch` apart, are no whole dwords
bool off_dwords(const int8_t* x, int64_t rows, int64_t K, int64_t pitch) {
  return ((K | (int64_t)reinterpret_cast<uintptr_t>(x) | (rows > 1 ? pitch : 0)) & 3) != 0;
}

// gemm_rcr_int8(a, b, a_scale, b_scale, bias, bf16, out, algo, workspace): bf16 is the result's type
PyObject* gemm_rcr_int8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    int64_t algo;
    if (nargs != 9 || !PyBool_Check(args[5]) || args[6] != Py_None || !number(args[7], &algo) || !plain_allocation()) return not_ordinary();
    const int dt = args[5] == Py_True ? 1 : 0;
    const at::ScalarType type = dt ? at::kBFloat16 : at::kHalf;
    Operands ops;
    const at::Tensor *a = ops.get(args[0], at::kChar), *b = ops.get(args[1], at::kChar), *a_scale = ops.get(args[2], at::kFloat),
                     *b_scale = ops.get(args[3], at::kFloat), *bias = ops.optional(args[4], type), *ws = ops.optional(args[8], at::kByte);
    if (!ops.ok || a->dim() < 1 || b->dim() != 2 || a->numel() == 0 || b->numel() == 0 || b->size(1) != a->size(-1)) return not_ordinary();
    const int64_t K = a->size(-1), N = b->size(0), M = a->numel() / K;
    int64_t lda, ldb;
    if (!flat_row_pitch(*a, M, K, &lda) || !row_pitch(*b, &ldb) || a_scale->numel() != M || !a_scale->is_contiguous() || b_scale->numel() != N ||
        !b_scale->is_contiguous() || (bias != nullptr && (bias->numel() != N || !bias->is_contiguous())) || (ws != nullptr && !ws->is_contiguous()))
      return not_ordinary();
    c10::SmallVector<int64_t, 6> sizes(a->sizes().begin(), a->sizes().end());
    sizes.back() = N;
    at::Tensor out = make(sizes, type, *a);
    const int8_t *pa = static_cast<const int8_t*>(a->data_ptr()), *pb = static_cast<const int8_t*>(b->data_ptr());
    at::Tensor scratch;  // (an operand whose rows are no whole dwords is laid out there first)
    const bool odd_a = off_dwords(pa, M, K, lda), odd_b = off_dwords(pb, N, K, ldb);
    if (ws == nullptr && algo < 0 && (odd_a || odd_b)) {
      const int64_t need = aitamd_gemm_int8_layout_bytes(odd_a ? M : 0, odd_b ? N : 0, K);
      if (need > 0) {
        scratch = make({need}, at::kByte, *a);
        ws = &scratch;
      }
    }
    const float *sa = static_cast<const float*>(a_scale->data_ptr()), *sb = static_cast<const float*>(b_scale->data_ptr());
    const void* pbias = pointer(bias);
    void *c = out.data_ptr(), *w = ws == nullptr ? nullptr : ws->data_ptr(), *stream = current_stream();
    const int64_t ws_bytes = ws == nullptr ? 0 : ws->numel();
    const int rc = unlocked([&] {
      return aitamd_gemm_rcr_int8(dt, (int)algo, pa, pb, sa, sb, pbias, c, M, N, K, lda, ldb, N, w, ws_bytes, stream);
    });
    return finish(rc, "gemm_rcr_int8", &out, nullptr);
  });
}

// rotary_embedding(x, positions, freqs, interleaved, scale, inverse, out)
PyObject* rotary_embedding(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    if (nargs != 7 || !PyBool_Check(args[3]) || !PyFloat_CheckExact(args[4]) || !PyBool_Check(args[5])) return not_ordinary();
    Operands ops;
    const at::Tensor* x;
    const int dt = first_operand(args[0], ops, &x);
    const at::Tensor* positions = gpu_tensor(args[1]);
    const at::Tensor* freqs = ops.get(args[2], at::kFloat);
    if (dt < 0 || !ops.ok || positions == nullptr || positions->device() != x->device() || x->numel() == 0 || !dense(*x)) return not_ordinary();
    const bool wide = positions->scalar_type() == at::kLong;
    const int64_t dims = x->dim();
    if ((!wide && positions->scalar_type() != at::kInt) || (dims != 3 && dims != 4) || freqs->dim() != 1 || !freqs->is_contiguous() ||
        2 * freqs->numel() > x->size(-1) || positions->dim() < 1 || positions->dim() > dims - 2 || positions->size(-1) != x->size(-3) ||
        (positions->dim() == 2 && positions->size(0) != x->size(0)))
      return not_ordinary();
    at::Tensor made;
    const at::Tensor* out = ops.optional(args[6], x->scalar_type());
    if (!ops.ok) return not_ordinary();
    if (out == nullptr) {
      if (!plain_allocation()) return not_ordinary();
      made = make(x->sizes(), x->scalar_type(), *x);
      out = &made;
    } else if (out->sizes() != x->sizes() || !dense(*out)) {
      return not_ordinary();
    }
    const bool flat = dims == 3;
    const int64_t batch = flat ? 1 : x->size(0), seq = x->size(-3), heads = x->size(-2), head_dim = x->size(-1), rotated = 2 * freqs->numel();
    const int64_t xb = flat ? 0 : x->stride(0), xs = x->stride(-3), xh = x->stride(-2), ob = flat ? 0 : out->stride(0), os = out->stride(-3),
                  oh = out->stride(-2), pb = positions->dim() == 2 ? positions->stride(0) : 0, ps = positions->stride(-1);
    const void *px = x->data_ptr(), *pp = positions->data_ptr();
    const float* pf = static_cast<const float*>(freqs->data_ptr());
    void *po = out->data_ptr(), *stream = current_stream();
    const float scale = (float)PyFloat_AS_DOUBLE(args[4]);
    const int interleaved = args[3] == Py_True, inverse = args[5] == Py_True;
    const int rc = unlocked([&] {
      return aitamd_rotary_embedding(dt, px, po, pp, wide, pf, batch, seq, heads, head_dim, rotated, xb, xs, xh, ob, os, oh, pb, ps, scale,
                                     interleaved, inverse, stream);
    });
    return finish(rc, "rotary_embedding", made.defined() ? &made : nullptr, args[6]);
  });
}

// a paged cache from (k_cache, v_cache, block_table, lengths, offsets) at args, for `tokens` rows of `head_dim`
bool paged_cache(PyObject* const* args, Operands& ops, at::ScalarType type, int64_t tokens, int64_t head_dim, aitamd_paged_cache* c) {
  const at::Tensor *k = ops.get(args[0], type), *v = ops.get(args[1], type), *table = ops.get(args[2], at::kInt),
                   *lengths = ops.get(args[3], at::kInt), *offsets = ops.optional(args[4], at::kInt);
  if (!ops.ok || k->dim() != 4 || v->sizes() != k->sizes() || k->size(3) != head_dim || !dense(*k) || !dense(*v) || lengths->dim() != 1 ||
      !lengths->is_contiguous())
    return false;
  const int64_t batch = lengths->numel();
  if (table->dim() != 2 || table->size(0) != batch || !dense(*table) ||
      (offsets != nullptr ? offsets->dim() != 1 || !offsets->is_contiguous() || offsets->numel() != batch + 1 : tokens != batch))
    return false;
  *c = {k->data_ptr(), v->data_ptr(), k->size(0), k->size(1), k->size(2), head_dim, k->stride(0), k->stride(1), k->stride(2), v->stride(0),
        v->stride(1), v->stride(2), static_cast<const int32_t*>(table->data_ptr()), table->stride(0), table->size(1),
        static_cast<const int32_t*>(lengths->data_ptr()), offsets == nullptr ? nullptr : static_cast<const int32_t*>(offsets->data_ptr()), batch,
        tokens};
  return true;
}

// the weights of `heads` heads' norms, of one or of each: false where they are no [head_dim] or [heads, head_dim]
bool norm_weight(const at::Tensor* w, int64_t heads, int64_t head_dim, const void** at, int64_t* stride) {
  *at = w == nullptr ? nullptr : w->data_ptr();
  *stride = 0;
  if (w == nullptr) return true;
  if (!dense(*w)) return false;
  if (w->dim() == 1) return w->size(0) == head_dim;
  if (w->dim() != 2 || w->size(0) != heads || w->size(1) != head_dim) return false;
  *stride = w->stride(0);
  return true;
}

// qk_norm_rotary(q, k, q_weight, k_weight, positions, freqs, eps, interleaved, scale, q_out, k_out): keys, frequencies and new results
PyObject* qk_norm_rotary(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    if (nargs != 11 || !PyFloat_CheckExact(args[6]) || !PyBool_Check(args[7]) || !PyFloat_CheckExact(args[8]) || args[9] != Py_None ||
        args[10] != Py_None || !plain_allocation())
      return not_ordinary();
    Operands ops;
    const at::Tensor* q;
    const int dt = first_operand(args[0], ops, &q);
    if (dt < 0 || q->numel() == 0 || !dense(*q)) return not_ordinary();
    const at::ScalarType type = q->scalar_type();
    const at::Tensor *k = ops.get(args[1], type), *q_weight = ops.optional(args[2], type), *k_weight = ops.optional(args[3], type),
                     *positions = gpu_tensor(args[4]), *freqs = ops.get(args[5], at::kFloat);
    if (!ops.ok || positions == nullptr || positions->device() != q->device()) return not_ordinary();
    const bool wide = positions->scalar_type() == at::kLong;
    const int64_t dims = q->dim();
    if ((!wide && positions->scalar_type() != at::kInt) || (dims != 3 && dims != 4) || freqs->dim() != 1 || !freqs->is_contiguous() ||
        2 * freqs->numel() > q->size(-1) || positions->dim() < 1 || positions->dim() > dims - 2 || positions->size(-1) != q->size(-3) ||
        (positions->dim() == 2 && positions->size(0) != q->size(0)) || k->dim() != dims || k->numel() == 0 || !dense(*k) ||
        k->size(-1) != q->size(-1) || k->size(-3) != q->size(-3) || (dims == 4 && k->size(0) != q->size(0)))
      return not_ordinary();
    const bool flat = dims == 3;
    const int64_t batch = flat ? 1 : q->size(0), seq = q->size(-3), head_dim = q->size(-1), rotated = 2 * freqs->numel();
    at::Tensor out[2] = {make(q->sizes(), type, *q), make(k->sizes(), type, *q)};
    aitamd_heads h[2];
    for (int i = 0; i < 2; ++i) {
      const at::Tensor &x = i ? *k : *q, &o = out[i];
      h[i] = {x.data_ptr(), o.data_ptr(), x.size(-2), flat ? 0 : x.stride(0), x.stride(-3), x.stride(-2), flat ? 0 : o.stride(0), o.stride(-3),
              o.stride(-2), nullptr, 0};
      if (!norm_weight(i ? k_weight : q_weight, x.size(-2), head_dim, &h[i].weight, &h[i].weight_head_stride)) return not_ordinary();
    }
    const int64_t pb = positions->dim() == 2 ? positions->stride(0) : 0, ps = positions->stride(-1);
    const void* pp = positions->data_ptr();
    const float *pf = static_cast<const float*>(freqs->data_ptr()), eps = (float)PyFloat_AS_DOUBLE(args[6]), scale = (float)PyFloat_AS_DOUBLE(args[8]);
    void* stream = current_stream();
    const int interleaved = args[7] == Py_True;
    const int rc = unlocked([&] {
      return aitamd_qk_norm_rotary(dt, &h[0], &h[1], pp, wide, pf, batch, seq, head_dim, rotated, pb, ps, eps, scale, interleaved, stream);
    });
    return pair_of(rc, "qk_norm_rotary", out[0], out[1]);
  });
}

// paged_kv_append(k, v, k_cache, v_cache, block_table, lengths, offsets, q, freqs, interleaved, scale, first_position, q_out): without
// frequencies the queries come back as they are.  With norms, (..., q_weight, k_weight, eps) behind that: of queries and keys that are
// turned
PyObject* append_rows(PyObject* const* args, bool normed) {
  return guarded([&]() -> PyObject* {
    int64_t first_position;
    if (!PyBool_Check(args[9]) || !PyFloat_CheckExact(args[10]) || !number(args[11], &first_position)) return not_ordinary();
    Operands ops;
    const at::Tensor* k;
    const int dt = first_operand(args[0], ops, &k);
    if (dt < 0 || k->dim() != 3 || k->numel() == 0) return not_ordinary();
    const at::ScalarType type = k->scalar_type();
    const at::Tensor *v = ops.get(args[1], type), *q = ops.optional(args[7], type), *freqs = ops.optional(args[8], at::kFloat),
                     *out = ops.optional(args[12], type);
    const int64_t tokens = k->size(0), head_dim = k->size(2);
    aitamd_paged_cache cache;
    if (!ops.ok || !paged_cache(args + 2, ops, type, tokens, head_dim, &cache) || cache.kv_heads != k->size(1) || v->sizes() != k->sizes() ||
        !dense(*k) || !dense(*v) ||
        (q != nullptr ? q->dim() != 3 || q->size(0) != tokens || q->size(2) != head_dim || q->numel() == 0 || !dense(*q) : out != nullptr) ||
        (freqs != nullptr ? freqs->dim() != 1 || !freqs->is_contiguous() || freqs->numel() == 0 || 2 * freqs->numel() > head_dim : out != nullptr))
      return not_ordinary();
    const bool turns = q != nullptr && freqs != nullptr;
    const void *q_weight = nullptr, *k_weight = nullptr;
    int64_t q_weight_head = 0, k_weight_head = 0;
    float eps = 0.0f;
    if (normed) {
      if (!turns || !PyFloat_CheckExact(args[15])) return not_ordinary();
      const at::Tensor *qw = ops.optional(args[13], type), *kw = ops.optional(args[14], type);
      if (!ops.ok || !norm_weight(qw, q->size(1), head_dim, &q_weight, &q_weight_head) ||
          !norm_weight(kw, k->size(1), head_dim, &k_weight, &k_weight_head))
        return not_ordinary();
      eps = (float)PyFloat_AS_DOUBLE(args[15]);
    }
    at::Tensor made;
    if (turns && out == nullptr) {
      if (!plain_allocation()) return not_ordinary();
      made = make(q->sizes(), type, *q);
      out = &made;
    } else if (turns && (out->sizes() != q->sizes() || !dense(*out))) {
      return not_ordinary();
    }
    const void *pk = k->data_ptr(), *pv = v->data_ptr(), *pq = turns ? q->data_ptr() : nullptr;
    void *po = turns ? out->data_ptr() : nullptr, *stream = current_stream();
    const float* pf = freqs == nullptr ? nullptr : static_cast<const float*>(freqs->data_ptr());
    const int64_t kt = k->stride(0), kh = k->stride(1), vt = v->stride(0), vh = v->stride(1), qt = turns ? q->stride(0) : 0,
                  qh = turns ? q->stride(1) : 0, ot = turns ? out->stride(0) : 0, oh = turns ? out->stride(1) : 0, heads = turns ? q->size(1) : 0,
                  rotated = freqs == nullptr ? 0 : 2 * freqs->numel();
    const float scale = (float)PyFloat_AS_DOUBLE(args[10]);
    const int interleaved = args[9] == Py_True;
    const int rc = unlocked([&] {
      return normed ? aitamd_paged_kv_append_norm(dt, &cache, pk, kt, kh, pv, vt, vh, pq, qt, qh, po, ot, oh, heads, q_weight, q_weight_head,
                                                  k_weight, k_weight_head, eps, pf, rotated, first_position, scale, interleaved, stream)
                    : aitamd_paged_kv_append(dt, &cache, pk, kt, kh, pv, vt, vh, pq, qt, qh, po, ot, oh, heads, pf, rotated, first_position,
                                             scale, interleaved, stream);
    });
    return finish(rc, "paged_kv_append", made.defined() ? &made : nullptr, turns ? args[12] : args[7]);
  });
}
PyObject* paged_kv_append(PyObject*, PyObject* const* args, Py_ssize_t nargs) { return nargs == 13 ? append_rows(args, false) : not_ordinary(); }
PyObject* paged_kv_append_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) { return nargs == 16 ? append_rows(args, true) : not_ordinary(); }

// prefix_attention(q, k_cache, v_cache, block_table, lengths, offsets, prefix_table, prefix_length, scale, out, workspace): a new
// result, a workspace of its own
PyObject* prefix_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    int64_t prefix;
    if (nargs != 11 || !number(args[7], &prefix) || !(args[8] == Py_None || PyFloat_CheckExact(args[8])) || !plain_allocation())
      return not_ordinary();
    Operands ops;
    const at::Tensor* q;
    const int dt = first_operand(args[0], ops, &q);
    if (dt < 0 || q->dim() != 3 || q->numel() == 0 || !dense(*q)) return not_ordinary();
    const int64_t tokens = q->size(0), heads = q->size(1), head_dim = q->size(2);
    aitamd_paged_cache cache;
    const at::Tensor *table = ops.optional(args[6], at::kInt), *out = ops.optional(args[9], q->scalar_type()), *ws = ops.optional(args[10], at::kByte);
    if (!ops.ok || !paged_cache(args + 1, ops, q->scalar_type(), tokens, head_dim, &cache) ||
        (table != nullptr ? table->dim() != 1 || !table->is_contiguous() : prefix != 0) ||
        (out != nullptr && (out->sizes() != q->sizes() || !dense(*out))) || (ws != nullptr && !ws->is_contiguous()))
      return not_ordinary();
    at::Tensor made, scratch;
    if (out == nullptr) {
      made = make(q->sizes(), q->scalar_type(), *q);
      out = &made;
    }
    if (ws == nullptr) {
      const int64_t need = aitamd_prefix_attention_workspace_bytes(&cache, heads, prefix);
      if (need > 0) {
        scratch = make({need}, at::kByte, *q);
        ws = &scratch;
      }
    }
    const void* pq = q->data_ptr();
    const int32_t* pt = table == nullptr ? nullptr : static_cast<const int32_t*>(table->data_ptr());
    void *po = out->data_ptr(), *w = ws == nullptr ? nullptr : ws->data_ptr(), *stream = current_stream();
    const int64_t qt = q->stride(0), qh = q->stride(1), ot = out->stride(0), oh = out->stride(1), pages = table == nullptr ? 0 : table->numel(),
                  ws_bytes = ws == nullptr ? 0 : ws->numel();
    const float scale = (float)(args[8] == Py_None ? std::pow((double)head_dim, -0.5) : PyFloat_AS_DOUBLE(args[8]));
    const int rc = unlocked([&] {
      return aitamd_prefix_attention(dt, &cache, pq, qt, qh, po, ot, oh, heads, pt, pages, prefix, scale, w, ws_bytes, stream);
    });
    return finish(rc, "prefix_attention", made.defined() ? &made : nullptr, args[9]);
  });
}

// gemm_rcr_lora(x, w, lora_a, lora_b, adapters, scales, bias, out, algo, workspace): a new result
PyObject* gemm_rcr_lora(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    int64_t algo;
    if (nargs != 10 || args[7] != Py_None || !number(args[8], &algo) || !plain_allocation()) return not_ordinary();
    Operands ops;
    const at::Tensor* x;
    const int dt = first_operand(args[0], ops, &x);
    if (dt < 0 || x->dim() < 1 || x->numel() == 0) return not_ordinary();
    const at::ScalarType type = x->scalar_type();
    const at::Tensor *w = ops.get(args[1], type), *a = ops.get(args[2], type), *b = ops.get(args[3], type), *of = ops.get(args[4], at::kInt),
                     *scales = ops.optional(args[5], at::kFloat), *bias = ops.optional(args[6], type), *ws = ops.optional(args[9], at::kByte);
    const int64_t K = x->size(-1), M = x->numel() / K;
    if (!ops.ok || w->dim() != 2 || w->numel() == 0 || w->size(1) != K || a->dim() != 3 || a->numel() == 0 || a->size(2) != K ||
        !a->is_contiguous() || b->dim() != 3 || !b->is_contiguous() || of->numel() != M || !of->is_contiguous())
      return not_ordinary();
    const int64_t N = w->size(0), n = a->size(0), rank = a->size(1);
    int64_t ldx, ldw;
    if (b->size(0) != n || b->size(1) != N || b->size(2) != rank || !flat_row_pitch(*x, M, K, &ldx) || !row_pitch(*w, &ldw) ||
        (scales != nullptr && (scales->numel() != n || !scales->is_contiguous())) ||
        (bias != nullptr && (bias->numel() != N || !bias->is_contiguous())) || (ws != nullptr && !ws->is_contiguous()))
      return not_ordinary();
    c10::SmallVector<int64_t, 6> sizes(x->sizes().begin(), x->sizes().end());
    sizes.back() = N;
    at::Tensor out = make(sizes, type, *x), scratch;
    if (ws == nullptr) {
      const int64_t need = aitamd_gemm_lora_workspace_bytes(dt, (int)algo, bias != nullptr, M, N, K, rank);
      scratch = make({std::max<int64_t>(need, 16)}, at::kByte, *x);
      ws = &scratch;
    }
    const void *px = x->data_ptr(), *pw = w->data_ptr(), *pa = a->data_ptr(), *pb = b->data_ptr(), *pbias = pointer(bias);
    const int32_t* po = static_cast<const int32_t*>(of->data_ptr());
    const float* ps = scales == nullptr ? nullptr : static_cast<const float*>(scales->data_ptr());
    void *c = out.data_ptr(), *scratch_at = ws->data_ptr(), *stream = current_stream();
    const int64_t ws_bytes = ws->numel();
    const int rc = unlocked([&] {
      return aitamd_gemm_rcr_lora(dt, (int)algo, px, pw, pbias, pa, pb, po, ps, c, M, N, K, rank, n, ldx, ldw, N, scratch_at, ws_bytes, stream);
    });
    return finish(rc, "gemm_rcr_lora", &out, nullptr);
  });
}

// token_logprobs(logits, tokens, top, scale, workspace)
PyObject* token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    int64_t top;
    if (nargs != 5 || !number(args[2], &top) || !PyFloat_CheckExact(args[3]) || top < 0 || !plain_allocation()) return not_ordinary();
    const at::Tensor *x = gpu_tensor(args[0]), *tokens = gpu_tensor(args[1]);
    if (x == nullptr || tokens == nullptr) return not_ordinary();
    Operands ops;
    const int dt = x->scalar_type() == at::kFloat ? (int)AITAMD_F32 : dtype_id(*x);
    const bool wide = tokens->scalar_type() == at::kLong;
    const at::Tensor* ws = ops.optional(args[4], at::kByte);
    if (dt < 0 || !ops.ok || !ops.here(*x) || !ops.here(*tokens) || (!wide && tokens->scalar_type() != at::kInt) || x->dim() < 1 || x->numel() == 0 ||
        !tokens->is_contiguous() || tokens->sizes() != x->sizes().slice(0, x->dim() - 1) || (ws != nullptr && !ws->is_contiguous()))
      return not_ordinary();
    const int64_t V = x->size(-1), rows = x->numel() / V;
    int64_t ld;
    if (!flat_row_pitch(*x, rows, V, &ld)) return not_ordinary();
    c10::SmallVector<int64_t, 6> sizes(x->sizes().begin(), x->sizes().end());
    sizes.back() = top;
    const at::IntArrayRef lead = x->sizes().slice(0, x->dim() - 1);
    at::Tensor made[5] = {make(lead, at::kFloat, *x), make(lead, at::kFloat, *x), make(lead, at::kInt, *x), make(sizes, at::kFloat, *x),
                          make(sizes, at::kInt, *x)};
    at::Tensor scratch;
    if (ws == nullptr) {
      const int64_t need = aitamd_token_logprobs_workspace_bytes(rows, V, top);
      if (need > 0) {
        scratch = make({need}, at::kByte, *x);
        ws = &scratch;
      }
    }
    const void *px = x->data_ptr(), *pt = tokens->data_ptr();
    float *lp = static_cast<float*>(made[0].data_ptr()), *en = static_cast<float*>(made[1].data_ptr()), *tl = static_cast<float*>(made[3].data_ptr());
    int32_t *rank = static_cast<int32_t*>(made[2].data_ptr()), *tt = static_cast<int32_t*>(made[4].data_ptr());
    void *w = ws == nullptr ? nullptr : ws->data_ptr(), *stream = current_stream();
    const int64_t ws_bytes = ws == nullptr ? 0 : ws->numel();
    const float scale = (float)PyFloat_AS_DOUBLE(args[3]);
    const int rc = unlocked([&] { return aitamd_token_logprobs(dt, px, pt, wide, lp, en, rank, tl, tt, rows, V, ld, top, scale, w, ws_bytes, stream); });
    if (rc != 0) return PyErr_Format(PyExc_RuntimeError, "token_logprobs failed: %s", aitamd_last_error());
    THPObjectPtr tuple(PyTuple_New(5));
    for (int i = 0; tuple && i < 5; ++i) {
      PyObject* o = THPVariable_Wrap(made[i]);
      if (o == nullptr) return nullptr;
      PyTuple_SET_ITEM(tuple.get(), i, o);
    }
    return tuple.release();
  });
}

PyMethodDef kMethods[] = {
#define AITAMD_METHOD(f, doc) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, doc}
    AITAMD_METHOD(quantize_rows, "quantize_rows(x)"),
    AITAMD_METHOD(gemm_rcr_int8, "gemm_rcr_int8(a, b, a_scale, b_scale, bias, bf16, out, algo, workspace)"),
    AITAMD_METHOD(rotary_embedding, "rotary_embedding(x, positions, freqs, interleaved, scale, inverse, out)"),
    AITAMD_METHOD(paged_kv_append,
                  "paged_kv_append(k, v, k_cache, v_cache, block_table, lengths, offsets, q, freqs, interleaved, scale, first_position, q_out)"),
    AITAMD_METHOD(paged_kv_append_norm,
                  "paged_kv_append_norm(k, v, k_cache, v_cache, block_table, lengths, offsets, q, freqs, interleaved, scale, first_position, "
                  "q_out, q_weight, k_weight, eps)"),
    AITAMD_METHOD(qk_norm_rotary, "qk_norm_rotary(q, k, q_weight, k_weight, positions, freqs, eps, interleaved, scale, q_out, k_out)"),
    AITAMD_METHOD(gemm_rcr_lora, "gemm_rcr_lora(x, w, lora_a, lora_b, adapters, scales, bias, out, algo, workspace)"),
    AITAMD_METHOD(token_logprobs, "token_logprobs(logits, tokens, top, scale, workspace)"),
    AITAMD_METHOD(prefix_attention,
                  "prefix_attention(q, k_cache, v_cache, block_table, lengths, offsets, prefix_table, prefix_length, scale, out, workspace)"),
#undef AITAMD_METHOD
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_native_decoder", "Eager calls of the decoder operators on torch tensors (see eager.py)", -1,
                       kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__native_decoder() {
  THPObjectPtr module(PyModule_Create(&kModule));
  if (!module || PyModule_AddStringConstant(module.get(), "torch_version", TORCH_VERSION) != 0 ||
      PyModule_AddStringConstant(module.get(), "torch_build", AITAMD_TORCH_BUILD) != 0)
    return nullptr;
  return module.release();
}
