// Compiled host path for torch callers: argument checks, output allocation and launches happen in C++, which takes the
// host cost of a call from 15 .. 70 us (Python + ctypes) to 4 .. 12 us -- small scales and small batches are bound by
// exactly that.  Two forms:
//   fast_*                            the operators of lvar_amd.sparse_attn_ops and the two steps of SparseDiffAttn for
//                                     well-formed inputs on the current device; every other input returns None and takes
//                                     the Python path, which raises the errors
//                                     (and of lvar_amd.kv_cache_ops, qk_norm_rope with its gradients)
//   register_dense_attn(ns)           defines and implements the torch-library op
//                                     `<ns>::dense_attn(Tensor q, Tensor k, Tensor v) -> Tensor[]`
//                                     natively, as the reference registers torch.ops.chipmunk.dense_attn
//                                     (kernels/chipmunk/csrc/chipmunk.cu:50-89, dense_attn at :57):
//                                     returns [o, 1/(2^M L)], softmax scale fixed to 1 (dense_attn.cu:161-163)
//
// The fast_* functions take their arguments as a C array (METH_FASTCALL) and allocate with torch's caching allocator
// directly: parsing through a signature and dispatching an `empty` would cost as much as the launch.
//
// The module does not link the C-ABI library: bind() receives the entry points' addresses from the Python
// side (which has loaded the library with ctypes), so both paths always call the same library.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <limits>
#include <memory>
#include <optional>
#include <string>
#include <vector>
#include <torch/extension.h>
#include <torch/library.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/custom_function.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include "../../include/lvar_sparse_attn.h"

namespace {

// entry points of the C-ABI library, by name
#define LVAR_ENTRIES(X)                                                                                                   \
  X(lvar_dense_attn_fwd) X(lvar_dense_attn_rcp_fwd) X(lvar_row_lse_scratch_bytes) X(lvar_row_lse_fwd)                     \
  X(lvar_lse2_from_stats) X(lvar_colsum_fwd) X(lvar_csp_attn_fwd) X(lvar_csp_attn_upsample_fwd)                           \
  X(lvar_csp_attn_remap_fwd)                                                                                              \
  X(lvar_block_sparse_attn_fwd) X(lvar_block_topk_lists) X(lvar_topk_token_lists) X(lvar_topk_union_lists)                \
  X(lvar_remap_concat_lists) X(lvar_mask_to_lists) X(lvar_window_key_scores)                                              \
  X(lvar_qk_norm_rope_fwd) X(lvar_qk_norm_rope_bwd_scratch_bytes) X(lvar_qk_norm_rope_bwd) X(lvar_kv_cache_append)        \
  X(lvar_kv_cache_read) X(lvar_paged_attn_workspace_bytes) X(lvar_paged_attn_fwd)
struct Api {
#define LVAR_FIELD(name) decltype(&::name) name = nullptr;
  LVAR_ENTRIES(LVAR_FIELD)
#undef LVAR_FIELD
} api;
bool bound = false;

std::vector<std::string> entry_names() {
  std::vector<std::string> v;
#define LVAR_NAME(name) v.emplace_back(#name);
  LVAR_ENTRIES(LVAR_NAME)
#undef LVAR_NAME
  return v;
}

// addresses in the order of entry_names()
void bind(const std::vector<uintptr_t>& a) {
  TORCH_CHECK(a.size() == entry_names().size(), "lvar_amd: wrong number of entry points");
  size_t i = 0;
#define LVAR_SET(name) api.name = reinterpret_cast<decltype(&::name)>(a[i++]);
  LVAR_ENTRIES(LVAR_SET)
#undef LVAR_SET
  bound = true;
}

bool plain(const at::Tensor& t) {
  return t.defined() && t.is_cuda() && t.dim() == 4 && t.scalar_type() == at::kBFloat16 && t.is_contiguous() &&
         (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
}

lvar_tensor_t view(const at::Tensor& t) {
  lvar_tensor_t v;
  v.ptr = t.data_ptr();
  v.stride_b = t.stride(0);
  v.stride_h = t.stride(1);
  v.stride_row = t.stride(2);
  return v;
}

// ---- argument helpers: each returns false / null for what the Python path has to look at ----
const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

// rows of a 4-d bf16 tensor that the kernels can read in place: unit stride on d, 16-byte aligned rows
bool rows_ok(const at::Tensor* t, int dev) {
  if (!t || !t->is_cuda() || t->get_device() != dev || t->dim() != 4 || t->scalar_type() != at::kBFloat16) return false;
  const auto st = t->strides();
  return st[3] == 1 && ((st[0] | st[1] | st[2]) & 7) == 0 && st[2] > 0 && (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15u) == 0;
}

// contiguous tensor of a dtype on the device
bool packed(const at::Tensor* t, int dev, at::ScalarType ty) {
  return t && t->is_cuda() && t->get_device() == dev && t->scalar_type() == ty && t->is_contiguous();
}

bool as_long(PyObject* o, int64_t& v) {
  if (!PyLong_CheckExact(o)) return false;
  v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) { PyErr_Clear(); return false; }
  return true;
}

bool as_bool(PyObject* o, bool& v) {
  if (!PyBool_Check(o)) return false;
  v = o == Py_True;
  return true;
}

bool as_double(PyObject* o, double& v) {
  if (PyFloat_CheckExact(o)) { v = PyFloat_AS_DOUBLE(o); return true; }
  int64_t i;
  if (!as_long(o, i)) return false;
  v = static_cast<double>(i);
  return true;
}

// softmax scale: None = 1/sqrt(d)
bool as_scale(PyObject* o, int64_t d, float& s) {
  if (o == Py_None) { s = static_cast<float>(1.0 / std::sqrt(static_cast<double>(d))); return true; }
  double v;
  if (!as_double(o, v)) return false;
  s = static_cast<float>(v);
  return true;
}

struct Qkv {
  const at::Tensor *q, *k, *v;
  int dev, B, H, Hkv, Lq, Lk, d;
  void* stream;
};

// q, k and (unless `v` is null) v of one attention call on the current device; `gqa`: fewer key heads than query heads
bool qkv_ok(Qkv& a, PyObject* q, PyObject* k, PyObject* v, bool gqa) {
  a.q = tensor(q); a.k = tensor(k); a.v = v ? tensor(v) : a.k;
  if (!bound || !a.q || !a.q->is_cuda()) return false;
  a.dev = a.q->get_device();
  if (!rows_ok(a.q, a.dev) || !rows_ok(a.k, a.dev) || !rows_ok(a.v, a.dev)) return false;
  const auto qs = a.q->sizes(), ks = a.k->sizes();
  if (a.v != a.k && a.v->sizes() != ks) return false;
  if (qs[0] != ks[0] || qs[3] != ks[3] || (qs[3] != 64 && qs[3] != 128 && qs[3] != 256)) return false;
  if (qs[0] <= 0 || qs[1] <= 0 || qs[2] <= 0 || ks[1] <= 0 || ks[2] <= 0 || qs[2] > INT32_MAX || ks[2] > INT32_MAX) return false;
  if (qs[1] != ks[1] && !(gqa && qs[1] % ks[1] == 0)) return false;
  if (c10::hip::current_device() != a.dev) return false;
  a.B = static_cast<int>(qs[0]); a.H = static_cast<int>(qs[1]); a.Hkv = static_cast<int>(ks[1]);
  a.Lq = static_cast<int>(qs[2]); a.Lk = static_cast<int>(ks[2]); a.d = static_cast<int>(qs[3]);
  a.stream = c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(a.dev)).stream();
  return true;
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType ty, int dev) {
  return at::Tensor(at::detail::empty_cuda(sizes, ty, at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(dev)), std::nullopt));
}
at::Tensor empty_o(const Qkv& a) { return empty({a.B, a.H, a.Lq, a.d}, at::kBFloat16, a.dev); }
at::Tensor empty_stat(const Qkv& a) { return empty({a.B, a.H, a.Lq, 1}, at::kFloat, a.dev); }

// M and L in one allocation: L is a view of the storage behind M
void empty_stats(const Qkv& a, at::Tensor& M, at::Tensor& L) {
  const int64_t rows = int64_t(a.B) * a.H * a.Lq;
  M = empty({2, a.B, a.H, a.Lq, 1}, at::kFloat, a.dev);
  L = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(M.storage()), M.key_set(), M.dtype());
  L.unsafeGetTensorImpl()->set_sizes_contiguous({a.B, a.H, a.Lq, 1});
  L.unsafeGetTensorImpl()->set_storage_offset(rows);
  M.unsafeGetTensorImpl()->set_sizes_contiguous({a.B, a.H, a.Lq, 1});
}

PyObject* none() { Py_RETURN_NONE; }

template <class... T>
PyObject* tuple(T&&... t) {
  PyObject* r = PyTuple_New(sizeof...(t));
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  (PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(std::forward<T>(t))), ...);
  return r;
}

#define LVAR_FAST(name) PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t n)
#define LVAR_NEED(cond) do { if (!(cond)) return none(); } while (0)

// (q, k, v, scale) -> (o, M, L)
LVAR_FAST(fast_dense_attn) {
  HANDLE_TH_ERRORS
  Qkv x;
  float scale;
  LVAR_NEED(n == 4 && qkv_ok(x, a[0], a[1], a[2], true) && as_scale(a[3], x.d, scale));
  at::Tensor o = empty_o(x), M, L;
  empty_stats(x, M, L);
  LVAR_NEED(api.lvar_dense_attn_fwd(view(*x.q), view(*x.k), view(*x.v), view(o), M.data_ptr<float>(), L.data_ptr<float>(), nullptr,
                                    x.B, x.H, x.Hkv, x.Lq, x.Lk, x.d, scale, x.stream) == LVAR_OK);
  return tuple(std::move(o), std::move(M), std::move(L));
  END_HANDLE_TH_ERRORS
}

int64_t groups_of(int64_t Lq, int64_t rows) { return (Lq + rows - 1) / rows; }

// (q, k, v, scale, group rows) -> (o, cs, M, L)
LVAR_FAST(fast_dense_colsum_attn) {
  HANDLE_TH_ERRORS
  Qkv x;
  float scale;
  int64_t bm;
  LVAR_NEED(n == 5 && qkv_ok(x, a[0], a[1], a[2], true) && as_scale(a[3], x.d, scale) && as_long(a[4], bm) && bm > 0 && bm % 32 == 0);
  at::Tensor o = empty_o(x), lse2 = empty_stat(x), M, L;
  empty_stats(x, M, L);
  at::Tensor cs = empty({x.B, x.H, groups_of(x.Lq, bm), x.Lk}, at::kFloat, x.dev);
  LVAR_NEED(api.lvar_dense_attn_fwd(view(*x.q), view(*x.k), view(*x.v), view(o), M.data_ptr<float>(), L.data_ptr<float>(), lse2.data_ptr<float>(),
                                    x.B, x.H, x.Hkv, x.Lq, x.Lk, x.d, scale, x.stream) == LVAR_OK);
  LVAR_NEED(api.lvar_colsum_fwd(view(*x.q), view(*x.k), lse2.data_ptr<float>(), cs.data_ptr<float>(), nullptr, x.B, x.H, x.Hkv, x.Lq, x.Lk, x.d,
                                static_cast<int>(bm), scale, x.stream) == LVAR_OK);
  return tuple(std::move(o), std::move(cs), std::move(M), std::move(L));
  END_HANDLE_TH_ERRORS
}

// (q, k, scale, group rows, M | None, L | None, want block sums, want columns) -> (cs | None, block sums | None)
LVAR_FAST(fast_colsum) {
  HANDLE_TH_ERRORS
  Qkv x;
  float scale;
  int64_t bm;
  bool want_bs, want_cs;
  LVAR_NEED(n == 8 && qkv_ok(x, a[0], a[1], nullptr, true) && as_scale(a[2], x.d, scale) && as_long(a[3], bm) && bm > 0 && bm % 32 == 0 &&
            as_bool(a[6], want_bs) && as_bool(a[7], want_cs) && (want_bs || want_cs));
  const bool given = a[4] != Py_None;
  const int64_t rows = int64_t(x.B) * x.H * x.Lq, G = groups_of(x.Lq, bm);
  const at::Tensor *M = nullptr, *L = nullptr;
  if (given) {
    M = tensor(a[4]); L = tensor(a[5]);
    LVAR_NEED(packed(M, x.dev, at::kFloat) && packed(L, x.dev, at::kFloat) && M->numel() == rows && L->numel() == rows);
  }
  at::Tensor lse2 = empty_stat(x), cs, bs;
  if (given) {
    LVAR_NEED(api.lvar_lse2_from_stats(M->data_ptr<float>(), L->data_ptr<float>(), lse2.data_ptr<float>(), rows, x.stream) == LVAR_OK);
  } else {
    // (block sums alone: the keys stay uncut, see _colsum_block_scores)
    const int64_t bytes = want_cs ? api.lvar_row_lse_scratch_bytes(x.B, x.H, x.Lq, x.Lk) : 0;
    at::Tensor scratch;
    if (bytes > 0) scratch = empty({bytes}, at::kByte, x.dev);
    LVAR_NEED(api.lvar_row_lse_fwd(view(*x.q), view(*x.k), lse2.data_ptr<float>(), bytes > 0 ? scratch.data_ptr() : nullptr, bytes > 0 ? bytes : 0,
                                   x.B, x.H, x.Hkv, x.Lq, x.Lk, x.d, scale, x.stream) == LVAR_OK);
  }
  if (want_cs) cs = empty({x.B, x.H, G, x.Lk}, at::kFloat, x.dev);
  if (want_bs) bs = empty({x.B, x.H, G, (x.Lk + 63) / 64}, at::kFloat, x.dev);
  LVAR_NEED(api.lvar_colsum_fwd(view(*x.q), view(*x.k), lse2.data_ptr<float>(), want_cs ? cs.data_ptr<float>() : nullptr,
                                want_bs ? bs.data_ptr<float>() : nullptr, x.B, x.H, x.Hkv, x.Lq, x.Lk, x.d, static_cast<int>(bm), scale, x.stream) == LVAR_OK);
  return tuple(std::move(cs), std::move(bs));   // (an undefined tensor wraps as None)
  END_HANDLE_TH_ERRORS
}

// key lists of a token-list call: int32, rows of one (batch, head) packed
bool lists_ok(const Qkv& x, const at::Tensor* idx, const at::Tensor* cnt, int64_t bm) {
  if (!idx || !packed(cnt, x.dev, at::kInt) || !idx->is_cuda() || idx->get_device() != x.dev || idx->scalar_type() != at::kInt) return false;
  if (idx->dim() != 4 || cnt->dim() != 3 || bm <= 0) return false;
  const auto s = idx->sizes(), st = idx->strides();
  if (s[0] != x.B || s[1] != x.H || s[2] <= 0 || s[2] > INT32_MAX || s[2] * bm < x.Lq) return false;
  if (cnt->size(0) != s[0] || cnt->size(1) != s[1] || cnt->size(2) != s[2]) return false;
  return st[3] == 1 && st[1] == s[2] * st[2] && st[0] == s[1] * st[1];
}

int csp_launch(const Qkv& x, const at::Tensor& idx, const at::Tensor& cnt, int64_t bm, const at::Tensor* accum, int up_src, int up_dst,
               const at::Tensor& o, float o_scale, float scale) {
  const lvar_tensor_t av = accum ? view(*accum) : lvar_tensor_t{};
  const int G = static_cast<int>(idx.size(2));
  if (up_src > 0)
    return api.lvar_csp_attn_upsample_fwd(view(*x.q), view(*x.k), view(*x.v), av, up_src, up_dst, view(o), nullptr, nullptr, idx.data_ptr<int32_t>(),
                                          cnt.data_ptr<int32_t>(), G, idx.stride(2), static_cast<int>(bm), x.B, x.H, x.Lq, x.Lk, x.d, o_scale, scale, x.stream);
  return api.lvar_csp_attn_fwd(view(*x.q), view(*x.k), view(*x.v), av, view(o), nullptr, nullptr, idx.data_ptr<int32_t>(), cnt.data_ptr<int32_t>(), G,
                               idx.stride(2), static_cast<int>(bm), x.B, x.H, x.Lq, x.Lk, x.d, o_scale, scale, x.stream);
}

// o_accum of a token-list call: shaped like q, or the coarse grid of `up_src` x `up_src` tokens
bool accum_ok(const Qkv& x, const at::Tensor* t, int64_t up_src, int64_t up_dst) {
  if (!rows_ok(t, x.dev) || t->size(0) != x.B || t->size(1) != x.H || t->size(3) != x.d) return false;
  return up_src > 0 ? (t->size(2) == up_src * up_src && up_dst * up_dst == x.Lq) : t->size(2) == x.Lq;
}

// (q, k, v, scale, indices, counts, o_accum, o_scale, group rows, up_src, up_dst) -> o
LVAR_FAST(fast_csp_attn) {
  HANDLE_TH_ERRORS
  Qkv x;
  float scale;
  double o_scale;
  int64_t bm, up_src, up_dst;
  LVAR_NEED(n == 11 && qkv_ok(x, a[0], a[1], a[2], false) && as_scale(a[3], x.d, scale) && as_double(a[7], o_scale) && as_long(a[8], bm) &&
            as_long(a[9], up_src) && as_long(a[10], up_dst) && up_src >= 0 && up_src < 32768 && up_dst < 32768);
  const at::Tensor *idx = tensor(a[4]), *cnt = tensor(a[5]), *acc = tensor(a[6]);
  LVAR_NEED(lists_ok(x, idx, cnt, bm) && idx->size(3) == x.Lk && accum_ok(x, acc, up_src, up_dst));
  at::Tensor o = empty_o(x);
  LVAR_NEED(csp_launch(x, *idx, *cnt, bm, acc, static_cast<int>(up_src), static_cast<int>(up_dst), o, static_cast<float>(o_scale), scale) == LVAR_OK);
  return THPVariable_Wrap(std::move(o));
  END_HANDLE_TH_ERRORS
}

// Decision-scale step of a column-sparse layer (models/sparvar/sparse_attn.py:991-1051): dense attention, column sums,
// top-k key lists and, if wanted, the output cache O - delta(O).
// (q, k, v, scale, group rows, keys per list, want cache) -> (o, indices, counts, cache | None)
LVAR_FAST(fast_full_step) {
  HANDLE_TH_ERRORS
  Qkv x;
  float scale;
  int64_t bm, keep;
  bool want_cache;
  LVAR_NEED(n == 7 && qkv_ok(x, a[0], a[1], a[2], false) && as_scale(a[3], x.d, scale) && as_long(a[4], bm) && bm > 0 && bm % 32 == 0 &&
            as_long(a[5], keep) && keep >= 0 && keep <= x.Lk && as_bool(a[6], want_cache));
  const int64_t G = groups_of(x.Lq, bm);
  at::Tensor o = empty_o(x), lse2 = empty_stat(x), cs = empty({x.B, x.H, G, x.Lk}, at::kFloat, x.dev);
  at::Tensor idx = empty({x.B, x.H, G, x.Lk}, at::kInt, x.dev), cnt = empty({x.B, x.H, G}, at::kInt, x.dev), cache;
  if (want_cache) cache = empty_o(x);
  LVAR_NEED(api.lvar_dense_attn_fwd(view(*x.q), view(*x.k), view(*x.v), view(o), nullptr, nullptr, lse2.data_ptr<float>(),
                                    x.B, x.H, x.Hkv, x.Lq, x.Lk, x.d, scale, x.stream) == LVAR_OK);
  LVAR_NEED(api.lvar_colsum_fwd(view(*x.q), view(*x.k), lse2.data_ptr<float>(), cs.data_ptr<float>(), nullptr, x.B, x.H, x.Hkv, x.Lq, x.Lk, x.d,
                                static_cast<int>(bm), scale, x.stream) == LVAR_OK);
  LVAR_NEED(api.lvar_topk_token_lists(cs.data_ptr<float>(), x.Lk, idx.data_ptr<int32_t>(), x.Lk, cnt.data_ptr<int32_t>(),
                                      static_cast<int>(int64_t(x.B) * x.H * G), x.Lk, static_cast<int>(keep), static_cast<int>(keep), x.stream) == LVAR_OK);
  if (want_cache) LVAR_NEED(csp_launch(x, idx, cnt, bm, &o, 0, 0, cache, -1.f, scale) == LVAR_OK);
  return tuple(std::move(o), std::move(idx), std::move(cnt), std::move(cache));
  END_HANDLE_TH_ERRORS
}

// key list of a sparse step: remapped decision-scale lists, then the local run (see remap_concat_lists)
bool remap(const at::Tensor& src, int64_t count, int64_t Gk, int64_t k_len, const at::Tensor* local, int64_t pad, int64_t out_len, bool zero_tail,
           int dev, void* stream, at::Tensor& idx, at::Tensor& cnt) {
  const int64_t B = src.size(0), H = src.size(1), Gs = src.size(2), Ks = src.size(3);
  const int64_t c = std::max(pad, (count + pad - 1) / pad * pad), L = local ? local->size(1) : 0;
  if (c + L > out_len || out_len > INT32_MAX) return false;
  idx = empty({B, H, Gk, out_len}, at::kInt, dev);
  cnt = empty({B, H, Gk}, at::kInt, dev);
  return api.lvar_remap_concat_lists(src.data_ptr<int32_t>(), Ks, static_cast<int>(Ks), local ? local->data_ptr<int64_t>() : nullptr, L, static_cast<int>(L),
                                     idx.data_ptr<int32_t>(), out_len, cnt.data_ptr<int32_t>(), static_cast<int>(B * H), static_cast<int>(Gs),
                                     static_cast<int>(Gk), static_cast<int>(c), static_cast<int>(k_len), static_cast<int>(zero_tail ? out_len : c + L), stream) == LVAR_OK;
}

// Step of a column-sparse layer after the decision scale (models/sparvar/sparse_attn.py:1053-1144): lists remapped to
// this scale's query groups + local run, then token-list attention on top of the upsampled output cache.
// Lists that no later step reads are not written (head_dim 64 and 128, groups of a multiple of 192 rows).
// (q, k, v, scale, src indices, src count, local, group rows, pad, cache, up_src, up_dst, keep lists) -> (o, indices | None, counts | None)
LVAR_FAST(fast_sparse_step) {
  HANDLE_TH_ERRORS
  Qkv x;
  float scale;
  int64_t count, bm, pad, up_src, up_dst;
  bool keep;
  LVAR_NEED(n == 13 && as_bool(a[12], keep) && qkv_ok(x, a[0], a[1], a[2], false) && as_scale(a[3], x.d, scale) && as_long(a[5], count) && as_long(a[7], bm) && bm > 0 &&
            as_long(a[8], pad) && pad > 0 && as_long(a[10], up_src) && as_long(a[11], up_dst) && up_src > 0 && up_src < 32768 && up_dst < 32768);
  const at::Tensor *src = tensor(a[4]), *local = tensor(a[6]), *cache = tensor(a[9]);
  const int64_t Gk = groups_of(x.Lq, bm);
  LVAR_NEED(packed(src, x.dev, at::kInt) && src->dim() == 4 && src->size(0) == x.B && src->size(1) == x.H && src->size(2) > 0 && count >= 0);
  LVAR_NEED(packed(local, x.dev, at::kLong) && local->dim() == 2 && local->size(0) == Gk && accum_ok(x, cache, up_src, up_dst));
  at::Tensor idx, cnt, o = empty_o(x);
  const int64_t c = std::max(pad, (count + pad - 1) / pad * pad), L = local->size(1), Ks = src->size(3);
  if (!keep && c <= Ks && c + L <= x.Lk) {
    const int st = api.lvar_csp_attn_remap_fwd(view(*x.q), view(*x.k), view(*x.v), view(*cache), static_cast<int>(up_src), static_cast<int>(up_dst), view(o),
                                               src->data_ptr<int32_t>(), Ks, static_cast<int>(Ks), static_cast<int>(src->size(2)), static_cast<int>(c),
                                               L > 0 ? local->data_ptr<int64_t>() : nullptr, L, static_cast<int>(L), static_cast<int>(bm), x.B, x.H, x.Lq,
                                               x.Lk, x.d, 1.f, scale, x.stream);
    if (st == LVAR_OK) return tuple(std::move(o), std::move(idx), std::move(cnt));
    LVAR_NEED(st == LVAR_EUNSUPPORTED);
  }
  LVAR_NEED(remap(*src, count, Gk, x.Lk, local, pad, x.Lk, false, x.dev, x.stream, idx, cnt));
  LVAR_NEED(csp_launch(x, idx, cnt, bm, cache, static_cast<int>(up_src), static_cast<int>(up_dst), o, 1.f, scale) == LVAR_OK);
  return tuple(std::move(o), std::move(idx), std::move(cnt));
  END_HANDLE_TH_ERRORS
}

// (q, k, v, kv_num_blocks, kv_indices, block_q, block_k, scale, want statistics) -> (o, M | None, L | None)
LVAR_FAST(fast_block_sparse_attn) {
  HANDLE_TH_ERRORS
  Qkv x;
  float scale;
  int64_t bq, bk;
  bool stats;
  LVAR_NEED(n == 9 && qkv_ok(x, a[0], a[1], a[2], false) && as_long(a[5], bq) && as_long(a[6], bk) && as_scale(a[7], x.d, scale) && as_bool(a[8], stats));
  LVAR_NEED((bq == 64 || (bq > 0 && bq % 128 == 0 && bq <= INT32_MAX)) && (bk == 64 || bk == 128 || bk == 256));
  const at::Tensor *num = tensor(a[3]), *idx = tensor(a[4]);
  LVAR_NEED(packed(num, x.dev, at::kInt) && packed(idx, x.dev, at::kInt) && num->dim() == 3 && idx->dim() == 4);
  const auto ns = num->sizes(), is = idx->sizes();
  const int64_t nQ = groups_of(x.Lq, bq);
  LVAR_NEED(ns[2] == nQ && is[2] == nQ && (ns[0] == 1 || ns[0] == x.B) && (ns[1] == 1 || ns[1] == x.H) && is[0] == ns[0] && is[1] == ns[1] &&
            is[3] > 0 && is[3] <= INT32_MAX);
  const bool per_b = ns[0] == x.B && x.B > 1, per_h = ns[1] == x.H && x.H > 1;
  at::Tensor o = empty_o(x), M, L;
  if (stats) empty_stats(x, M, L);
  LVAR_NEED(api.lvar_block_sparse_attn_fwd(view(*x.q), view(*x.k), view(*x.v), view(o), stats ? M.data_ptr<float>() : nullptr, stats ? L.data_ptr<float>() : nullptr,
                                           num->data_ptr<int32_t>(), per_b ? num->stride(0) : 0, per_h ? num->stride(1) : 0, idx->data_ptr<int32_t>(),
                                           per_b ? idx->stride(0) : 0, per_h ? idx->stride(1) : 0, is[3], static_cast<int>(is[3]), static_cast<int>(bq),
                                           static_cast<int>(bk), x.B, x.H, x.Lq, x.Lk, x.d, scale, x.stream) == LVAR_OK);
  return tuple(std::move(o), std::move(M), std::move(L));
  END_HANDLE_TH_ERRORS
}

// device and stream of a list-building call: `t` lives on the current device
bool list_call(const at::Tensor* t, int& dev, void*& stream) {
  if (!bound || !t || !t->is_cuda()) return false;
  dev = t->get_device();
  if (c10::hip::current_device() != dev) return false;
  stream = c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(dev)).stream();
  return true;
}

// (block scores, target, base mask | None) -> (kv_num_blocks, kv_indices)
LVAR_FAST(fast_block_topk_lists) {
  HANDLE_TH_ERRORS
  const at::Tensor* s = n == 3 ? tensor(a[0]) : nullptr;
  int dev;
  void* stream;
  int64_t target;
  LVAR_NEED(list_call(s, dev, stream) && packed(s, dev, at::kFloat) && s->dim() == 4 && s->numel() > 0 && as_long(a[1], target) && target >= 0 && target <= INT32_MAX);
  const int64_t B = s->size(0), H = s->size(1), nQ = s->size(2), nK = s->size(3);
  const at::Tensor* base = a[2] == Py_None ? nullptr : tensor(a[2]);
  if (a[2] != Py_None) LVAR_NEED(base && base->dim() == 2 && base->size(0) == nQ && base->size(1) == nK && (packed(base, dev, at::kBool) || packed(base, dev, at::kByte)));
  LVAR_NEED(nK <= 2048 && B * H * nQ <= INT32_MAX);
  at::Tensor num = empty({B, H, nQ}, at::kInt, dev), idx = empty({B, H, nQ, nK}, at::kInt, dev);
  LVAR_NEED(api.lvar_block_topk_lists(s->data_ptr<float>(), base ? static_cast<const uint8_t*>(base->data_ptr()) : nullptr, num.data_ptr<int32_t>(),
                                      idx.data_ptr<int32_t>(), static_cast<int>(B), static_cast<int>(H), static_cast<int>(nQ), static_cast<int>(nK),
                                      static_cast<int>(target), stream) == LVAR_OK);
  return tuple(std::move(num), std::move(idx));
  END_HANDLE_TH_ERRORS
}

// (scores, k, out_len, zero_tail) -> (indices, counts)
LVAR_FAST(fast_topk_token_lists) {
  HANDLE_TH_ERRORS
  const at::Tensor* s = n == 4 ? tensor(a[0]) : nullptr;
  int dev;
  void* stream;
  int64_t k, out_len;
  bool zero_tail;
  LVAR_NEED(list_call(s, dev, stream) && packed(s, dev, at::kFloat) && s->dim() >= 1 && s->numel() > 0 && as_long(a[1], k) && as_long(a[2], out_len) && as_bool(a[3], zero_tail));
  const int64_t n_col = s->size(-1), rows = s->numel() / n_col;
  LVAR_NEED(k >= 0 && k <= n_col && out_len >= k && out_len <= INT32_MAX && rows <= INT32_MAX && n_col <= INT32_MAX);
  std::vector<int64_t> shape = s->sizes().vec();
  shape.back() = out_len;
  at::Tensor idx = empty(shape, at::kInt, dev);
  shape.pop_back();
  at::Tensor cnt = empty(shape, at::kInt, dev);
  LVAR_NEED(api.lvar_topk_token_lists(s->data_ptr<float>(), n_col, idx.data_ptr<int32_t>(), out_len, cnt.data_ptr<int32_t>(), static_cast<int>(rows),
                                      static_cast<int>(n_col), static_cast<int>(k), static_cast<int>(zero_tail ? out_len : k), stream) == LVAR_OK);
  return tuple(std::move(idx), std::move(cnt));
  END_HANDLE_TH_ERRORS
}

// (src indices, src count, query groups, k_len, local | None, pad, out_len, zero_tail) -> (indices, counts)
LVAR_FAST(fast_remap_concat_lists) {
  HANDLE_TH_ERRORS
  const at::Tensor* src = n == 8 ? tensor(a[0]) : nullptr;
  int dev;
  void* stream;
  int64_t count, Gk, k_len, pad, out_len;
  bool zero_tail;
  LVAR_NEED(list_call(src, dev, stream) && packed(src, dev, at::kInt) && src->dim() == 4 && src->numel() > 0 && as_long(a[1], count) && as_long(a[2], Gk) &&
            as_long(a[3], k_len) && as_long(a[5], pad) && as_long(a[6], out_len) && as_bool(a[7], zero_tail) && count >= 0 && Gk > 0 && pad > 0 && k_len > 0);
  const at::Tensor* local = a[4] == Py_None ? nullptr : tensor(a[4]);
  if (a[4] != Py_None) LVAR_NEED(packed(local, dev, at::kLong) && local->dim() == 2 && local->size(0) == Gk);
  at::Tensor idx, cnt;
  LVAR_NEED(remap(*src, count, Gk, k_len, local, pad, out_len, zero_tail, dev, stream, idx, cnt));
  return tuple(std::move(idx), std::move(cnt));
  END_HANDLE_TH_ERRORS
}

// (bool mask, multiple) -> (counts, indices)
LVAR_FAST(fast_mask_to_lists) {
  HANDLE_TH_ERRORS
  const at::Tensor* m = n == 2 ? tensor(a[0]) : nullptr;
  int dev;
  void* stream;
  int64_t mult;
  LVAR_NEED(list_call(m, dev, stream) && packed(m, dev, at::kBool) && m->dim() >= 1 && m->numel() > 0 && as_long(a[1], mult) && mult > 0 && mult <= INT32_MAX);
  const int64_t n_col = m->size(-1), rows = m->numel() / n_col;
  LVAR_NEED(n_col <= INT32_MAX && rows <= INT32_MAX);
  at::Tensor idx = empty(m->sizes(), at::kInt, dev), cnt = empty(m->sizes().slice(0, m->dim() - 1), at::kInt, dev);
  LVAR_NEED(api.lvar_mask_to_lists(static_cast<const uint8_t*>(m->data_ptr()), n_col, idx.data_ptr<int32_t>(), n_col, cnt.data_ptr<int32_t>(),
                                   static_cast<int>(rows), static_cast<int>(n_col), static_cast<int>(mult), stream) == LVAR_OK);
  return tuple(std::move(cnt), std::move(idx));
  END_HANDLE_TH_ERRORS
}

// (q, k, window keys, pool kernel size, max pool, scale, keep) -> keep > 0: the kept positions, int64 [B,H,keep+W], the
// `keep` best-scoring keys and the window keys in ascending order; keep = 0: the scores, fp32 [B,H,Lk]
LVAR_FAST(fast_window_keys) {
  HANDLE_TH_ERRORS
  Qkv x;
  float scale;
  int64_t ksize, keep;
  bool maxpool;
  LVAR_NEED(n == 7 && qkv_ok(x, a[0], a[1], nullptr, false) && as_long(a[3], ksize) && as_bool(a[4], maxpool) && as_scale(a[5], x.d, scale) && as_long(a[6], keep));
  const at::Tensor* win = tensor(a[2]);
  LVAR_NEED(packed(win, x.dev, at::kLong) && win->dim() == 3 && win->size(0) == x.B && win->size(1) == x.H && win->size(2) > 0 && win->size(2) <= 65535);
  LVAR_NEED(x.Lq <= x.Lk && ksize % 2 == 1 && ksize >= 1 && ksize <= 33 && keep >= 0 && keep <= x.Lk);
  const int W = static_cast<int>(win->size(2));
  if (keep > 0) LVAR_NEED(x.Lk <= 16384);
  at::Tensor scores = empty({x.B, x.H, x.Lk}, at::kFloat, x.dev), out;
  if (keep > 0) out = empty({x.B, x.H, keep + W}, at::kLong, x.dev);
  LVAR_NEED(api.lvar_window_key_scores(view(*x.q), view(*x.k), win->data_ptr<int64_t>(), W, scores.data_ptr<float>(), x.B, x.H, x.Lq, x.Lk, x.d,
                                       static_cast<int>(ksize), maxpool ? 1 : 0, scale, x.stream) == LVAR_OK);
  if (keep == 0) return THPVariable_Wrap(std::move(scores));
  LVAR_NEED(api.lvar_topk_union_lists(scores.data_ptr<float>(), x.Lk, win->data_ptr<int64_t>(), W, out.data_ptr<int64_t>(), x.B * x.H, x.Lk,
                                      static_cast<int>(keep), x.stream) == LVAR_OK);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---- norms with rotation, the paged cache, attention over it (lvar_amd.kv_cache_ops) ----

// a tensor or None; false: neither
bool optional_tensor(PyObject* o, const at::Tensor*& t) {
  t = o == Py_None ? nullptr : tensor(o);
  return o == Py_None || t;
}

bool wants_grad(const at::Tensor* t) { return t && t->requires_grad() && at::GradMode::is_enabled(); }
// a forward-mode derivative, which no operator here has (the Python path raises)
bool has_tangent(const at::Tensor* t) { return t && t->_fw_grad(0).defined(); }
bool wants_derivative(const at::Tensor* t) { return wants_grad(t) || has_tangent(t); }

// int32 [B] on the device, or nothing
bool per_sequence(const at::Tensor* t, int64_t B, int dev) { return !t || (packed(t, dev, at::kInt) && t->dim() == 1 && t->size(0) == B); }
const int32_t* ints(const at::Tensor* t) { return t ? t->data_ptr<int32_t>() : nullptr; }

bool same_strides(const at::Tensor& a, const at::Tensor& b, int64_t dims) {
  for (int64_t i = 0; i < dims; i++)
    if (a.size(i) != b.size(i) || (a.size(i) > 1 && a.stride(i) != b.stride(i))) return false;
  return true;
}

// cache: the tuple (k, v, k_exp, v_exp) (the entry points check alignments and limits)
bool cache_ok(PyObject* cache, PyObject* page_table, int64_t B, int dev, lvar_paged_cache_t& c) {
  if (!PyTuple_Check(cache) || PyTuple_GET_SIZE(cache) != 4) return false;
  PyObject* const a[4] = {PyTuple_GET_ITEM(cache, 0), PyTuple_GET_ITEM(cache, 1), PyTuple_GET_ITEM(cache, 2), PyTuple_GET_ITEM(cache, 3)};
  const at::Tensor *k = tensor(a[0]), *v = tensor(a[1]), *table = tensor(page_table), *ke, *ve;
  if (!k || !v || !table || !optional_tensor(a[2], ke) || !optional_tensor(a[3], ve)) return false;
  const bool f8 = k->scalar_type() == at::kFloat8_e4m3fn;
  if ((!f8 && k->scalar_type() != at::kBFloat16) || v->scalar_type() != k->scalar_type() || k->dim() != 4 || v->dim() != 4) return false;
  if (wants_derivative(k) || wants_derivative(v)) return false;
  if (!k->is_cuda() || k->get_device() != dev || !v->is_cuda() || v->get_device() != dev || !same_strides(*k, *v, 4)) return false;
  if (k->stride(3) != 1 || v->stride(3) != 1 || k->numel() == 0) return false;
  for (int i = 0; i < 4; i++) if (k->size(i) > INT32_MAX) return false;
  c = {};
  if (f8) {
    if (!ke || !ve) return false;
    for (const at::Tensor* e : {ke, ve}) {
      if (!e->is_cuda() || e->get_device() != dev || e->scalar_type() != at::kByte || e->dim() != 3 || e->stride(2) != 1) return false;
      for (int i = 0; i < 3; i++) if (e->size(i) != k->size(i)) return false;
    }
    if (!same_strides(*ke, *ve, 3)) return false;
    c.k_exp = ke->data_ptr<uint8_t>(); c.v_exp = ve->data_ptr<uint8_t>();
    c.exp_stride_page = ke->size(0) > 1 ? ke->stride(0) : 0; c.exp_stride_head = ke->size(1) > 1 ? ke->stride(1) : 0;
  } else if (ke || ve) {
    return false;
  }
  if (!table->is_cuda() || table->get_device() != dev || table->scalar_type() != at::kInt || table->dim() != 2 || table->size(0) != B ||
      table->size(1) <= 0 || table->size(1) > INT32_MAX || (table->stride(1) != 1 && table->size(1) > 1))
    return false;
  c.k = k->data_ptr(); c.v = v->data_ptr();
  c.stride_page = k->size(0) > 1 ? k->stride(0) : 0; c.stride_head = k->size(1) > 1 ? k->stride(1) : 0; c.stride_row = k->stride(2);
  c.page_table = table->data_ptr<int32_t>(); c.table_stride = B > 1 ? table->stride(0) : 0;
  c.num_pages = static_cast<int>(k->size(0)); c.kv_heads = static_cast<int>(k->size(1)); c.page_size = static_cast<int>(k->size(2));
  c.head_dim = static_cast<int>(k->size(3)); c.max_pages = static_cast<int>(table->size(1));
  return true;
}

// The tensors of a cache (as cache_ok takes it) have been written: autograd finds out where it has saved them; tensors of inference mode have no version.
void count_write(PyObject* cache) {
  for (int i = 0; i < 4; i++) {
    const at::Tensor* t = tensor(PyTuple_GET_ITEM(cache, i));
    if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  }
}

bool weight_ok(const at::Tensor* w, int64_t heads, int64_t d, int dev, lvar_weight_t& v) {
  v = {};
  if (!w) return true;
  if (!w->is_cuda() || w->get_device() != dev || (w->scalar_type() != at::kFloat && w->scalar_type() != at::kBFloat16)) return false;
  const int64_t n = w->dim(), rows = n == 2 ? w->size(0) : 1, cols = n == 2 ? w->size(1) : n == 1 ? w->size(0) : 0;
  if ((n != 1 && n != 2) || (rows != 1 && rows != heads) || (cols != d && (cols != 1 || n == 1))) return false;
  if ((rows > 1 && w->stride(0) == 0) || (cols > 1 && w->stride(n - 1) != 1)) return false;
  v.ptr = w->data_ptr(); v.stride_head = rows > 1 ? w->stride(0) : 0; v.stride_col = cols > 1 ? 1 : 0; v.dtype = w->scalar_type() == at::kBFloat16;
  return true;
}

// what a call says about the norm and the rotation, apart from the weights
struct How {
  lvar_norm_rope_t h;
  const at::Tensor *cos, *sin, *positions;
};

// a: cos, sin, positions, q_weight, k_weight, norm, eps, interleaved
bool how_ok(PyObject* const* a, const at::Tensor& q, const at::Tensor& k, int dev, bool needs_rows, How& w, const at::Tensor*& wq, const at::Tensor*& wk) {
  const int64_t B = q.size(0), L = q.size(2), d = q.size(3);
  w.h = {};
  if (!optional_tensor(a[0], w.cos) || !optional_tensor(a[1], w.sin) || !optional_tensor(a[2], w.positions) || !optional_tensor(a[3], wq) || !optional_tensor(a[4], wk)) return false;
  if (a[5] == Py_None) { w.h.norm = LVAR_NORM_NONE; w.h.eps = 0.f; }
  else if (PyUnicode_Check(a[5]) && PyUnicode_CompareWithASCIIString(a[5], "l2") == 0) { w.h.norm = LVAR_NORM_L2; w.h.eps = 1e-12f; }
  else if (PyUnicode_Check(a[5]) && PyUnicode_CompareWithASCIIString(a[5], "rms") == 0) { w.h.norm = LVAR_NORM_RMS; w.h.eps = 1e-6f; }
  else return false;
  double eps;
  bool inter;
  if (a[6] != Py_None) { if (!as_double(a[6], eps) || (eps != 0.0 && !(eps >= std::numeric_limits<float>::min()))) return false; w.h.eps = static_cast<float>(eps); }
  if (!as_bool(a[7], inter)) return false;
  if (!w.cos != !w.sin) return false;
  if (w.cos) {
    for (const at::Tensor* t : {w.cos, w.sin})
      if (!t->is_cuda() || t->get_device() != dev || t->scalar_type() != at::kFloat || t->dim() != 2 || t->stride(1) != 1 || t->requires_grad() ||
          has_tangent(t))
        return false;
    if (w.cos->sizes() != w.sin->sizes() || w.cos->stride(0) != w.sin->stride(0) || w.cos->size(0) <= 0 || w.cos->size(0) > INT32_MAX || 2 * w.cos->size(1) > d) return false;
    if (needs_rows && !w.positions && w.cos->size(0) < L) return false;
    w.h.cos = w.cos->data_ptr<float>(); w.h.sin = w.sin->data_ptr<float>(); w.h.table_stride = w.cos->stride(0);
    w.h.table_rows = static_cast<int>(w.cos->size(0)); w.h.rot_dim = static_cast<int>(2 * w.cos->size(1)); w.h.interleaved = inter;
  }
  if (w.positions) {
    const at::Tensor& p = *w.positions;
    const int64_t n = p.dim();
    if (!p.is_cuda() || p.get_device() != dev || (p.scalar_type() != at::kInt && p.scalar_type() != at::kLong)) return false;
    if ((n != 1 && n != 2) || p.size(n - 1) != L || (n == 2 && p.size(0) != B)) return false;
    w.h.positions = p.data_ptr(); w.h.positions64 = p.scalar_type() == at::kLong;
    w.h.pos_stride_b = n == 2 && B > 1 ? p.stride(0) : 0; w.h.pos_stride_row = p.stride(n - 1);
  }
  return weight_ok(wq, q.size(1), d, dev, w.h.q_weight) && weight_ok(wk, k.size(1), d, dev, w.h.k_weight);
}

// q and k of a norm on the current device
bool qk_ok(const at::Tensor* q, const at::Tensor* k, int& dev, void*& stream) {
  if (!bound || !q || !k || !q->is_cuda()) return false;
  dev = q->get_device();
  if (!rows_ok(q, dev) || !rows_ok(k, dev) || q->numel() == 0 || k->numel() == 0) return false;
  if (q->size(0) != k->size(0) || q->size(2) != k->size(2) || q->size(3) != k->size(3) || q->size(1) % k->size(1) != 0) return false;
  for (int i = 0; i < 3; i++) if (q->size(i) > INT32_MAX) return false;
  if (c10::hip::current_device() != dev) return false;
  stream = c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(dev)).stream();
  return true;
}

int dim(const at::Tensor& t, int i) { return static_cast<int>(t.size(i)); }

int norm_rope_launch(const at::Tensor& q, const at::Tensor& k, const lvar_norm_rope_t& h, at::Tensor& oq, at::Tensor& ok, int dev, void* stream) {
  oq = empty(q.sizes(), at::kBFloat16, dev);
  ok = empty(k.sizes(), at::kBFloat16, dev);
  return api.lvar_qk_norm_rope_fwd(view(q), view(k), h, oq.data_ptr(), ok.data_ptr(), dim(q, 0), dim(q, 1), dim(k, 1), dim(q, 2), dim(q, 3), stream);
}

// memory for a gradient of t in t's own order of axes, if the kernels can write it
at::Tensor rows_like(const at::Tensor& t) {
  at::Tensor g = t.is_non_overlapping_and_dense() ? at::Tensor(at::detail::empty_strided_cuda(t.sizes(), t.strides(), at::kBFloat16, t.device())) : at::empty_like(t);
  const auto st = g.strides();
  return st[3] == 1 && ((st[0] | st[1] | st[2]) & 7) == 0 ? g : at::empty(t.sizes(), t.options());
}

// The C call's arguments that are not tensors travel in `h`; its pointers are set anew from the saved tensors.
struct NormRopeFunction : torch::autograd::Function<NormRopeFunction> {
  using Maybe = std::optional<at::Tensor>;   // (undefined tensors are no inputs)
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const Maybe& wq,
                                                const Maybe& wk, const Maybe& cos, const Maybe& sin, const Maybe& positions, const lvar_norm_rope_t* h,
                                                int64_t stream) {
    auto some = [](const Maybe& t) { return t.value_or(at::Tensor()); };
    ctx->save_for_backward({q, k, some(wq), some(wk), some(cos), some(sin), some(positions)});
    ctx->saved_data["how"] = std::string(reinterpret_cast<const char*>(h), sizeof(*h));
    at::Tensor oq, ok;
    const int st = norm_rope_launch(q, k, *h, oq, ok, q.get_device(), reinterpret_cast<void*>(stream));
    TORCH_CHECK(st == LVAR_OK, "lvar_qk_norm_rope_fwd failed with status ", st);
    return {oq, ok};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "qk_norm_rope can be differentiated once: its gradients have no graph (create_graph)");
    TORCH_CHECK(!has_tangent(&grads[0]) && !has_tangent(&grads[1]), "the gradient of qk_norm_rope has no forward-mode derivative: call it on tensors without a tangent");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &q = saved[0], &k = saved[1], &wq = saved[2], &wk = saved[3], &cos = saved[4], &sin = saved[5], &positions = saved[6];
    lvar_norm_rope_t h;
    const std::string how = ctx->saved_data["how"].toStringRef();
    std::memcpy(&h, how.data(), sizeof(h));
    // (pointers and strides anew: hooks on saved tensors may return copies of another layout)
    const int dev = q.get_device(), B = dim(q, 0), H = dim(q, 1), Hkv = dim(k, 1), L = dim(q, 2), d = dim(q, 3);
    auto ptr = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    auto there = [](const at::Tensor& t) { return t.defined() ? &t : nullptr; };
    bool same = rows_ok(&q, dev) && rows_ok(&k, dev) && weight_ok(there(wq), H, d, dev, h.q_weight) && weight_ok(there(wk), Hkv, d, dev, h.k_weight);
    if (cos.defined()) {
      same = same && cos.is_cuda() && sin.is_cuda() && cos.get_device() == dev && sin.get_device() == dev && cos.stride(1) == 1 && sin.stride(1) == 1 && cos.stride(0) == sin.stride(0);
      h.cos = cos.data_ptr<float>(); h.sin = sin.data_ptr<float>(); h.table_stride = cos.stride(0);
    }
    if (positions.defined()) {
      same = same && positions.is_cuda() && positions.get_device() == dev;
      h.positions = positions.data_ptr();
      h.pos_stride_b = positions.dim() == 2 && B > 1 ? positions.stride(0) : 0; h.pos_stride_row = positions.stride(-1);
    }
    TORCH_CHECK(same, "qk_norm_rope: hooks on saved tensors returned tensors that the backward pass cannot read (device, alignment or strides)");
    const c10::DeviceGuard guard(q.device());
    auto rows = [](const at::Tensor& g) {
      at::Tensor c = g.contiguous();
      return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) ? c.clone() : c;
    };
    const at::Tensor gq = rows(grads[0]), gk = rows(grads[1]);
    at::Tensor dq = rows_like(q), dk = rows_like(k), dwq, dwk, scratch;
    if (wq.defined() && wq.requires_grad()) dwq = empty(wq.sizes(), wq.scalar_type(), dev);
    if (wk.defined() && wk.requires_grad()) dwk = empty(wk.sizes(), wk.scalar_type(), dev);
    int64_t bytes = 0;
    if (dwq.defined() || dwk.defined()) {
      bytes = api.lvar_qk_norm_rope_bwd_scratch_bytes(B, H, Hkv, L, d);
      if (bytes > 0) scratch = empty({bytes}, at::kByte, dev);
    }
    const int st = api.lvar_qk_norm_rope_bwd(view(q), view(k), h, gq.data_ptr(), gk.data_ptr(), view(dq), view(dk), ptr(dwq), ptr(dwk), ptr(scratch), bytes, B, H,
                                             Hkv, L, d, c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(dev)).stream());
    TORCH_CHECK(st == LVAR_OK, "lvar_qk_norm_rope_bwd failed with status ", st);
    return {dq, dk, dwq, dwk, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// (q, k, cos, sin, positions, q_weight, k_weight, norm, eps, interleaved) -> (q, k)
LVAR_FAST(fast_qk_norm_rope) {
  HANDLE_TH_ERRORS
  const at::Tensor *q = n == 10 ? tensor(a[0]) : nullptr, *k = n == 10 ? tensor(a[1]) : nullptr, *wq, *wk;
  int dev;
  void* stream;
  How w;
  LVAR_NEED(qk_ok(q, k, dev, stream) && how_ok(a + 2, *q, *k, dev, true, w, wq, wk));
  LVAR_NEED(!has_tangent(q) && !has_tangent(k) && !has_tangent(wq) && !has_tangent(wk));
  at::Tensor oq, ok;
  if (wants_grad(q) || wants_grad(k) || wants_grad(wq) || wants_grad(wk)) {
    // (declined before a graph is built: what the entry point would refuse raises in the Python path)
    LVAR_NEED(std::isfinite(w.h.eps) && w.h.eps >= 0.f && (!w.cos || (w.h.rot_dim % 16 == 0 && w.h.rot_dim > 0 && w.h.table_stride % 4 == 0 &&
              ((reinterpret_cast<uintptr_t>(w.h.cos) | reinterpret_cast<uintptr_t>(w.h.sin)) & 15u) == 0)));
    for (const auto* x : {&w.h.q_weight, &w.h.k_weight})
      LVAR_NEED(!x->stride_col || ((reinterpret_cast<uintptr_t>(x->ptr) & 15u) == 0 && x->stride_head % 8 == 0));
    const int64_t d = q->size(3);
    LVAR_NEED((d == 16 || d == 32 || d == 64 || d == 128 || d == 256) && q->size(0) <= 65535 && q->size(1) <= 16384 && q->size(0) * q->size(2) <= (1ll << 30));
    auto some = [](const at::Tensor* t) { return t ? std::optional<at::Tensor>(*t) : std::nullopt; };
    auto r = NormRopeFunction::apply(*q, *k, some(wq), some(wk), some(w.cos), some(w.sin), some(w.positions), &w.h, reinterpret_cast<int64_t>(stream));
    return tuple(std::move(r[0]), std::move(r[1]));
  }
  LVAR_NEED(norm_rope_launch(*q, *k, w.h, oq, ok, dev, stream) == LVAR_OK);
  return tuple(std::move(oq), std::move(ok));
  END_HANDLE_TH_ERRORS
}

// (cache, page table, start, counts, q | None, k, v[, cos, sin, positions, q_weight, k_weight, norm, eps, interleaved]) -> q, or True
LVAR_FAST(fast_kv_append) {
  HANDLE_TH_ERRORS
  LVAR_NEED(n == 7 || n == 15);
  const bool fused = n == 15;
  const at::Tensor *q = fused ? tensor(a[4]) : tensor(a[5]), *k = tensor(a[5]), *v = tensor(a[6]), *start = tensor(a[2]), *counts, *wq = nullptr, *wk = nullptr;
  int dev;
  void* stream;
  LVAR_NEED(qk_ok(q, k, dev, stream) && rows_ok(v, dev) && v->sizes() == k->sizes() && start && optional_tensor(a[3], counts));
  const int64_t B = k->size(0);
  lvar_paged_cache_t c;
  LVAR_NEED(per_sequence(start, B, dev) && per_sequence(counts, B, dev) && cache_ok(a[0], a[1], B, dev, c) && c.kv_heads == k->size(1) && c.head_dim == k->size(3));
  How w;
  if (fused) LVAR_NEED(how_ok(a + 7, *q, *k, dev, false, w, wq, wk));
  LVAR_NEED(!wants_derivative(q) && !wants_derivative(k) && !wants_derivative(v) && !wants_derivative(wq) && !wants_derivative(wk));
  at::Tensor oq;
  if (fused) oq = empty(q->sizes(), at::kBFloat16, dev);
  LVAR_NEED(api.lvar_kv_cache_append(view(*q), view(*k), view(*v), fused ? &w.h : nullptr, fused ? oq.data_ptr() : nullptr, c, ints(start), ints(counts),
                                     static_cast<int>(B), dim(*q, 1), dim(*k, 2), stream) == LVAR_OK);
  count_write(a[0]);
  if (!fused) Py_RETURN_TRUE;
  return THPVariable_Wrap(std::move(oq));
  END_HANDLE_TH_ERRORS
}

// a length bound: None = everything that the table can name
bool as_bound(PyObject* o, const lvar_paged_cache_t& c, bool clamp, int64_t& v) {
  const int64_t reach = static_cast<int64_t>(c.max_pages) * c.page_size;
  if (o == Py_None) v = reach;
  else if (!as_long(o, v)) return false;
  if (clamp) v = std::min(v, reach);
  return v >= 0 && v <= INT32_MAX;
}

// (cache, page table, lengths, max_len, start) -> (k, v)
LVAR_FAST(fast_kv_read) {
  HANDLE_TH_ERRORS
  const at::Tensor *k = n == 5 && PyTuple_Check(a[0]) && PyTuple_GET_SIZE(a[0]) == 4 ? tensor(PyTuple_GET_ITEM(a[0], 0)) : nullptr, *table = n == 5 ? tensor(a[1]) : nullptr, *start;
  LVAR_NEED(bound && k && table && k->is_cuda() && table->dim() == 2 && optional_tensor(a[4], start));
  const int dev = k->get_device();
  const int64_t B = table->size(0);
  const at::Tensor* lengths = tensor(a[2]);
  lvar_paged_cache_t c;
  int64_t most;
  LVAR_NEED(lengths && c10::hip::current_device() == dev && cache_ok(a[0], a[1], B, dev, c) && per_sequence(lengths, B, dev) && per_sequence(start, B, dev) &&
            as_bound(a[3], c, false, most) && most > 0 && B > 0 && B <= 65535);
  at::Tensor ko = empty({B, c.kv_heads, most, c.head_dim}, at::kBFloat16, dev), vo = empty({B, c.kv_heads, most, c.head_dim}, at::kBFloat16, dev);
  LVAR_NEED(api.lvar_kv_cache_read(c, ints(start), ints(lengths), ko.data_ptr(), vo.data_ptr(), static_cast<int>(B), static_cast<int>(most),
                                   c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(dev)).stream()) == LVAR_OK);
  return tuple(std::move(ko), std::move(vo));
  END_HANDLE_TH_ERRORS
}

// (q, cache, page table, lengths, counts, scale, causal, max_len) -> (o, M, L)
LVAR_FAST(fast_paged_attn) {
  HANDLE_TH_ERRORS
  const at::Tensor *q = n == 8 ? tensor(a[0]) : nullptr, *counts;
  LVAR_NEED(bound && q && q->is_cuda());
  Qkv x{};
  x.dev = q->get_device();
  LVAR_NEED(rows_ok(q, x.dev) && q->numel() > 0 && c10::hip::current_device() == x.dev && !wants_derivative(q) && optional_tensor(a[4], counts));
  for (int i = 0; i < 3; i++) LVAR_NEED(q->size(i) <= INT32_MAX);
  x.B = dim(*q, 0); x.H = dim(*q, 1); x.Lq = dim(*q, 2); x.d = dim(*q, 3);
  const at::Tensor* lengths = tensor(a[3]);
  lvar_paged_cache_t c;
  float scale;
  bool causal;
  int64_t most;
  LVAR_NEED(lengths && cache_ok(a[1], a[2], x.B, x.dev, c) && c.head_dim == x.d && x.H % c.kv_heads == 0 && per_sequence(lengths, x.B, x.dev) &&
            per_sequence(counts, x.B, x.dev) && as_scale(a[5], x.d, scale) && as_bool(a[6], causal) && as_bound(a[7], c, true, most));
  const int64_t bytes = api.lvar_paged_attn_workspace_bytes(x.B, x.H, c.kv_heads, x.Lq, static_cast<int>(most), x.d);
  LVAR_NEED(bytes >= 0);
  at::Tensor o = empty_o(x), M, L, ws;
  empty_stats(x, M, L);
  if (bytes > 0) ws = empty({bytes}, at::kByte, x.dev);
  LVAR_NEED(api.lvar_paged_attn_fwd(view(*q), c, ints(lengths), ints(counts), o.data_ptr(), M.data_ptr<float>(), L.data_ptr<float>(), bytes > 0 ? ws.data_ptr() : nullptr,
                                    bytes, x.B, x.H, x.Lq, static_cast<int>(most), causal ? 1 : 0, scale,
                                    c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(x.dev)).stream()) == LVAR_OK);
  return tuple(std::move(o), std::move(M), std::move(L));
  END_HANDLE_TH_ERRORS
}

// rows are read with 16-byte accesses: anything else is copied into a plain tensor first
at::Tensor as_plain(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() == 4, name, " must be [B,H,L,d], got ", t.sizes());
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be bfloat16, got ", t.scalar_type());
  TORCH_CHECK(t.is_cuda(), name, " must live on a HIP device; lvar_amd has no CPU path");
  if (plain(t)) return t;
  at::Tensor c = t.contiguous();
  if (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) c = c.clone();
  return c;
}

// <ns>::dense_attn(q, k, v) -> [o, 1/(2^M L)]
std::vector<at::Tensor> op_dense_attn(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in) {
  TORCH_CHECK(bound, "lvar_amd: the C-ABI library is not bound");
  const at::Tensor q = as_plain(q_in, "q"), k = as_plain(k_in, "k"), v = as_plain(v_in, "v");
  const int64_t B = q.size(0), H = q.size(1), Lq = q.size(2), d = q.size(3), Lk = k.size(2);
  TORCH_CHECK(k.sizes() == v.sizes(), "k/v shape mismatch: ", k.sizes(), " vs ", v.sizes());
  const int64_t Hkv = k.size(1);
  TORCH_CHECK(k.size(0) == B && Hkv > 0 && H % Hkv == 0 && k.size(3) == d, "q/k batch, head or head_dim mismatch: ", q.sizes(), " vs ", k.sizes());
  TORCH_CHECK(q.get_device() == k.get_device() && q.get_device() == v.get_device(), "q, k, v must be on the same device");
  TORCH_CHECK(Lq <= INT32_MAX && Lk <= INT32_MAX, "sequence too long");
  const c10::DeviceGuard guard(q.device());   // the tensors' device is current for the allocations and the launch
  at::Tensor o = at::empty_like(q);
  at::Tensor rcp = at::empty({B, H, Lq, 1}, q.options().dtype(at::kFloat));
  void* stream = c10::hip::getCurrentHIPStream(q.get_device()).stream();
  const int st = api.lvar_dense_attn_rcp_fwd(view(q), view(k), view(v), view(o), rcp.data_ptr<float>(), static_cast<int>(B), static_cast<int>(H), static_cast<int>(Hkv),
                             static_cast<int>(Lq), static_cast<int>(Lk), static_cast<int>(d), 1.0f, stream);
  TORCH_CHECK(st == LVAR_OK, "lvar_dense_attn_rcp_fwd failed with status ", st,
              st == LVAR_EUNSUPPORTED ? " (unsupported head_dim)" : st == LVAR_EINVAL ? " (invalid argument)" : " (launch failed)");
  return {o, rcp};
}

// Libraries registered by register_dense_attn live until the process ends (as a TORCH_LIBRARY block's would).
std::vector<std::unique_ptr<torch::Library>>& libraries() {
  static std::vector<std::unique_ptr<torch::Library>> libs;
  return libs;
}

void register_dense_attn(const std::string& ns) {
  auto lib = std::make_unique<torch::Library>(torch::Library::FRAGMENT, ns, std::nullopt, __FILE__, __LINE__);
  lib->def("dense_attn(Tensor q, Tensor k, Tensor v) -> Tensor[]");
  lib->impl("dense_attn", torch::dispatch(c10::DispatchKey::CUDA, TORCH_FN(op_dense_attn)));
  libraries().push_back(std::move(lib));
}

#define LVAR_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef fast_methods[] = {
    LVAR_METHOD(fast_dense_attn), LVAR_METHOD(fast_dense_colsum_attn), LVAR_METHOD(fast_colsum), LVAR_METHOD(fast_csp_attn),
    LVAR_METHOD(fast_full_step), LVAR_METHOD(fast_sparse_step), LVAR_METHOD(fast_block_sparse_attn), LVAR_METHOD(fast_block_topk_lists),
    LVAR_METHOD(fast_topk_token_lists), LVAR_METHOD(fast_remap_concat_lists), LVAR_METHOD(fast_mask_to_lists), LVAR_METHOD(fast_window_keys),
    LVAR_METHOD(fast_qk_norm_rope), LVAR_METHOD(fast_kv_append), LVAR_METHOD(fast_kv_read), LVAR_METHOD(fast_paged_attn),
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("entry_names", &entry_names, "names of the C-ABI entry points that bind() takes the addresses of");
  m.def("bind", &bind);
  m.def("register_dense_attn", &register_dense_attn, "define and implement <ns>::dense_attn natively");
  if (PyModule_AddFunctions(m.ptr(), fast_methods) != 0) throw pybind11::error_already_set();
}
