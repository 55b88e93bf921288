// The eager calls of the paged cache and the log probabilities without Python's
// share of their cost: the checks of shard_amd/ops.py, the outputs' and the
// workspace's allocation and the call, for operands as programs pass them.
// Whatever is not plain (other types, layouts that need a copy, another device
// than the current one, refusals) returns None here and takes the way through
// ops.py, which copies or says what is wrong.
//
// Host time of a call beside one MI355X, launches included, us, here / through
// ops.py: kv4_append with q 4.8 / 10.1, kv4_read 5.3 / 8.4, kv4_attn (two launches)
// 8.1 / 13.5, token_logprobs (two launches) 9.0 / 16.5, kv4_tree_attn 8.6 / 15.2,
// verify_drafts 8.2 / 16.6, draft_tree, kv4_append and kv4_keep together 27-30 / 43.
#include <Python.h>
#include <dlfcn.h>

#include <algorithm>
#include <cmath>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/Allocator.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/shard_hip.h"

namespace {

decltype(&shard_kv4_append) p_append;
decltype(&shard_kv4_read) p_read;
decltype(&shard_kv4_attn_workspace) p_attn_workspace;
decltype(&shard_kv4_attn) p_attn;
decltype(&shard_token_logprobs_workspace) p_logprobs_workspace;
decltype(&shard_token_logprobs) p_logprobs;
// null where the library has none of them: their calls go through ops.py
decltype(&shard_kv4_append_at) p_append_at;
decltype(&shard_kv4_tree_attn_workspace) p_tree_workspace;
decltype(&shard_kv4_tree_attn) p_tree_attn;
decltype(&shard_kv4_keep) p_keep;
decltype(&shard_draft_tree) p_tree;
decltype(&shard_verify_drafts_workspace) p_verify_workspace;
decltype(&shard_verify_drafts) p_verify;

// Uninitialized, on like's device (the current one); without the dispatcher's
// share of at::empty (0.47 us against 0.71).
at::Tensor make(at::IntArrayRef size, const at::Tensor& like, at::ScalarType type) {
  return at::detail::empty_cuda(size, type, like.device(), std::nullopt);
}
c10::DataPtr scratch(size_t bytes) {  // of the current device and stream, given back when it goes out of scope
  return bytes ? c10::GetAllocator(c10::DeviceType::CUDA)->allocate(bytes) : c10::DataPtr();
}

// Other Python threads run while this one allocates and launches (a launch waits
// where the stream's queue is full, an allocation where it reaches the driver).
// No Python object is made or looked at within; operands stay alive, the caller
// holds them.
class Unlocked {
 public:
  Unlocked() : state(PyEval_SaveThread()) {}
  ~Unlocked() { PyEval_RestoreThread(state); }
  Unlocked(const Unlocked&) = delete;
  Unlocked& operator=(const Unlocked&) = delete;

 private:
  PyThreadState* state;
};

// A tensor argument on the current device; `none`: may be None (then null).
bool tensor(PyObject* o, int64_t device, const at::Tensor** t, bool none = false) {
  *t = nullptr;
  if (o == Py_None) return none;
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& x = THPVariable_Unpack(o);
  if (!x.is_cuda() || x.layout() != at::kStrided || x.get_device() != device) return false;
  *t = &x;
  return true;
}
bool integer(PyObject* o, int64_t* v) {  // None: 0
  if (o == Py_None) {
    *v = 0;
    return true;
  }
  if (!PyLong_Check(o)) return false;
  int overflow = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow == 0;
}
bool hint(PyObject* o, int32_t* v) {
  int64_t x;
  if (!integer(o, &x) || x < 0 || x > INT32_MAX) return false;
  *v = (int32_t)x;
  return true;
}

int half_code(const at::Tensor& t) {
  return t.scalar_type() == at::kHalf ? SHARD_FP16 : t.scalar_type() == at::kBFloat16 ? SHARD_BF16 : -1;
}

// n whole numbers of 32 bits, one after the other.
bool indexes(const at::Tensor& t, int64_t n) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}

// The batch's part of an argument block (_kv4_batch of ops.py); `d`: the cache's
// dimensions before the pages.
bool batch(shard_kv4_args& a, int64_t n_tokens, const at::Tensor& cache, const at::Tensor& table, const at::Tensor& lens,
           const at::Tensor* cu, int d = 0) {
  if (cache.dim() != 3 + d || table.dim() != 2 || lens.dim() != 1 || cache.scalar_type() != at::kByte || table.scalar_type() != at::kInt ||
      lens.scalar_type() != at::kInt)
    return false;
  const int64_t pages = cache.size(d), G = cache.size(d + 1), width = cache.size(d + 2), B = table.size(0), W = table.size(1);
  if ((width != 68 * 64 && width != 68 * 128) || lens.size(0) != B || !lens.is_contiguous()) return false;
  if (cu ? !indexes(*cu, B + 1) : n_tokens != B) return false;
  if (cache.stride(d + 2) != 1 || (cache.stride(d + 1) != width && G > 1) || (table.stride(1) != 1 && W > 1)) return false;
  const int64_t s0 = pages == 1 ? G * width : cache.stride(d), t0 = B == 1 ? W : table.stride(0);
  if (pages <= 0 || G <= 0 || W <= 0 || B <= 0 || s0 < G * width || t0 < W || n_tokens <= 0) return false;
  if (pages > INT32_MAX || G > INT32_MAX || W > INT32_MAX || B > INT32_MAX || n_tokens > INT32_MAX) return false;
  a.batch = (int32_t)B;
  a.n_tokens = (int32_t)n_tokens;
  a.n_kv_heads = (int32_t)G;
  a.head_dim = (int32_t)(width / 68);
  a.n_pages = (int32_t)pages;
  a.table_width = (int32_t)W;
  a.cache = (uint8_t*)cache.data_ptr();
  a.page_stride = s0;
  a.block_table = (const int32_t*)table.data_ptr();
  a.table_stride = t0;
  a.seq_lens = (const int32_t*)lens.data_ptr();
  a.cu_seqlens = cu ? (const int32_t*)cu->data_ptr() : nullptr;
  return true;
}

// A (tokens, heads, head_dim) operand that needs no copy (_kv4_rows of ops.py).
bool rows(const at::Tensor& t, int64_t n_tokens, int64_t heads, int64_t D, const void** p, int64_t* s0, int64_t* s1) {
  if (t.dim() != 3 || t.size(0) != n_tokens || t.size(2) != D || (heads && t.size(1) != heads)) return false;
  *s0 = t.stride(0);
  *s1 = t.stride(1);
  *p = t.data_ptr();
  return t.stride(2) == 1 && ((*s0 | *s1) & 7) == 0 && ((uintptr_t)*p & 15) == 0;
}

// kv4_append(k, v, cache, block_table, seq_lens, phases, q, cu_seqlens, max_new, [positions,] device, stream) -> rotated q, or True
PyObject* append(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t device, stream;
  const at::Tensor *k, *v, *cache, *table, *lens, *phases, *q, *cu, *at;
  shard_kv4_args a{};
  if ((n != 11 && n != 12) || !integer(o[n - 2], &device) || !integer(o[n - 1], &stream) || !tensor(o[0], device, &k) || !tensor(o[1], device, &v) ||
      !tensor(o[2], device, &cache) || !tensor(o[3], device, &table) || !tensor(o[4], device, &lens) || !tensor(o[5], device, &phases) ||
      !tensor(o[6], device, &q, true) || !tensor(o[7], device, &cu, true) || !hint(o[8], &a.max_new) ||
      !tensor(n == 12 ? o[9] : Py_None, device, &at, true) || (at && !p_append_at))
    Py_RETURN_NONE;
  if (k->dim() != 3 || !batch(a, k->size(0), *cache, *table, *lens, cu) || (at && !indexes(*at, a.n_tokens))) Py_RETURN_NONE;
  a.dtype = half_code(*k);
  const int64_t D = a.head_dim;
  if (a.dtype < 0 || v->scalar_type() != k->scalar_type() || (q && q->scalar_type() != k->scalar_type())) Py_RETURN_NONE;
  if (!rows(*k, a.n_tokens, a.n_kv_heads, D, &a.k, &a.k_stride, &a.k_head_stride) ||
      !rows(*v, a.n_tokens, a.n_kv_heads, D, &a.v, &a.v_stride, &a.v_head_stride))
    Py_RETURN_NONE;
  if (phases->scalar_type() != at::kFloat || phases->dim() != 3 || phases->size(1) != D / 2 || phases->size(2) != 2 ||
      !phases->is_contiguous() || ((uintptr_t)phases->data_ptr() & 15) || phases->size(0) < (int64_t)SHARD_KV4_PAGE * a.table_width ||
      phases->size(0) > INT32_MAX)
    Py_RETURN_NONE;
  a.phases = (const float*)phases->data_ptr();
  a.n_phases = (int32_t)phases->size(0);
  if (q) {
    if (!rows(*q, a.n_tokens, 0, D, &a.q, &a.q_stride, &a.q_head_stride) || q->size(1) <= 0 || q->size(1) > INT32_MAX) Py_RETURN_NONE;
    a.n_q_heads = (int32_t)q->size(1);
  }
  at::Tensor out;
  int rc;
  {
    const Unlocked unlocked;
    if (q) {
      out = make(q->sizes(), *q, q->scalar_type());
      a.q_out = out.data_ptr();
    }
    rc = at ? p_append_at(&a, (const int32_t*)at->data_ptr(), (void*)stream) : p_append(&a, (void*)stream);
  }
  if (rc) Py_RETURN_NONE;
  if (!q) Py_RETURN_TRUE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// kv4_read(cache, block_table, seq_lens, n_tokens, bf16, cu_seqlens, max_new, device, stream) -> k, v
PyObject* read(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t device, stream, n_tokens;
  const at::Tensor *cache, *table, *lens, *cu;
  shard_kv4_args a{};
  if (n != 9 || !integer(o[7], &device) || !integer(o[8], &stream) || !integer(o[3], &n_tokens) || !tensor(o[0], device, &cache) ||
      !tensor(o[1], device, &table) || !tensor(o[2], device, &lens) || !tensor(o[5], device, &cu, true) || !hint(o[6], &a.max_new) ||
      !batch(a, n_tokens, *cache, *table, *lens, cu))
    Py_RETURN_NONE;
  const bool bf16 = o[4] == Py_True;
  a.dtype = bf16 ? SHARD_BF16 : SHARD_FP16;
  const int64_t size[3] = {a.n_tokens, a.n_kv_heads, a.head_dim};
  const auto type = bf16 ? at::kBFloat16 : at::kHalf;
  at::Tensor k, v;
  int rc;
  {
    const Unlocked unlocked;
    k = make(size, *cache, type);
    v = make(size, *cache, type);
    a.k_out = k.data_ptr();
    a.v_out = v.data_ptr();
    rc = p_read(&a, (void*)stream);
  }
  if (rc) Py_RETURN_NONE;
  return Py_BuildValue("NN", THPVariable_Wrap(std::move(k)), THPVariable_Wrap(std::move(v)));
  END_HANDLE_TH_ERRORS
}

// kv4_attn(q, cache, block_table, seq_lens, cu_seqlens, scale, max_new, max_len, device, stream) -> out
// kv4_tree_attn(q, cache, block_table, seq_lens, cu_seqlens, scale, max_new, max_len, mask, device, stream) -> out
PyObject* attn(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t device, stream;
  const at::Tensor *q, *cache, *table, *lens, *cu, *mask;
  shard_kv4_args a{};
  if ((n != 10 && n != 11) || !integer(o[n - 2], &device) || !integer(o[n - 1], &stream) || !tensor(o[0], device, &q) || !tensor(o[1], device, &cache) ||
      !tensor(o[2], device, &table) || !tensor(o[3], device, &lens) || !tensor(o[4], device, &cu, true) || !hint(o[6], &a.max_new) ||
      !hint(o[7], &a.max_len) || !tensor(n == 11 ? o[8] : Py_None, device, &mask, n == 10) || (mask && !p_tree_attn))
    Py_RETURN_NONE;
  if (q->dim() != 3 || !batch(a, q->size(0), *cache, *table, *lens, cu)) Py_RETURN_NONE;
  a.dtype = half_code(*q);
  if (a.dtype < 0 || !rows(*q, a.n_tokens, 0, a.head_dim, &a.q, &a.q_stride, &a.q_head_stride)) Py_RETURN_NONE;
  const int64_t H = q->size(1);
  if (H <= 0 || H > INT32_MAX || H % a.n_kv_heads) Py_RETURN_NONE;
  a.n_q_heads = (int32_t)H;
  if (o[5] == Py_None) a.scale = (float)std::pow((double)a.head_dim, -0.5);
  else if (PyFloat_CheckExact(o[5])) a.scale = (float)PyFloat_AS_DOUBLE(o[5]);
  else Py_RETURN_NONE;
  if (mask && (mask->scalar_type() != at::kLong || mask->dim() != 2 || mask->size(0) != a.n_tokens || mask->size(1) < 1 ||
               mask->size(1) > INT32_MAX || !mask->is_contiguous()))
    Py_RETURN_NONE;
  at::Tensor out;
  int rc;
  {
    const Unlocked unlocked;
    out = make(q->sizes(), *q, q->scalar_type());
    a.out = out.data_ptr();
    const size_t need = mask ? p_tree_workspace(&a) : p_attn_workspace(&a);
    const c10::DataPtr ws = scratch(need);
    rc = mask ? p_tree_attn(&a, (const uint64_t*)mask->data_ptr(), (int32_t)mask->size(1), ws.get(), need, (void*)stream)
              : p_attn(&a, ws.get(), need, (void*)stream);
  }
  if (rc) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// A tree's bound (_tree_width of ops.py).
bool tree_width(PyObject* o, int64_t rows, int64_t* width) {
  if (o == Py_None) *width = rows;
  else if (!integer(o, width)) return false;
  *width = std::min(*width, rows);
  if (*width < 0 || *width > SHARD_TREE_ROWS) return false;
  *width = std::max<int64_t>(*width, 1);
  return true;
}

// draft_tree(parents, seq_lens, cu_seqlens, max_new, device, stream) -> mask, positions
PyObject* tree(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t device, stream, width;
  const at::Tensor *up, *lens, *cu;
  if (!p_tree || n != 6 || !integer(o[4], &device) || !integer(o[5], &stream) || !tensor(o[0], device, &up) || !tensor(o[1], device, &lens) ||
      !tensor(o[2], device, &cu, true) || up->dim() != 1 || lens->dim() != 1)
    Py_RETURN_NONE;
  const int64_t T = up->size(0), B = lens->size(0);
  if (T <= 0 || T > INT32_MAX || B <= 0 || B > INT32_MAX || !indexes(*up, T) || !indexes(*lens, B) ||
      (cu ? !indexes(*cu, B + 1) : T != B) || !tree_width(o[3], T, &width))
    Py_RETURN_NONE;
  const int64_t two[2] = {T, (width + 63) / 64}, one[1] = {T};
  at::Tensor mask, positions;
  int rc;
  {
    const Unlocked unlocked;
    mask = make(two, *up, at::kLong);
    positions = make(one, *up, at::kInt);
    rc = p_tree((const int32_t*)up->data_ptr(), (const int32_t*)lens->data_ptr(), cu ? (const int32_t*)cu->data_ptr() : nullptr,
                (int32_t)B, (int32_t)T, (int32_t)two[1], (uint64_t*)mask.data_ptr(), (int32_t*)positions.data_ptr(), (void*)stream);
  }
  if (rc) Py_RETURN_NONE;
  return Py_BuildValue("NN", THPVariable_Wrap(std::move(mask)), THPVariable_Wrap(std::move(positions)));
  END_HANDLE_TH_ERRORS
}

// kv4_keep(cache, block_table, seq_lens, rows, counts, cu_seqlens, device, stream) -> True
PyObject* keep(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t device, stream;
  const at::Tensor *cache, *table, *lens, *rows, *counts, *cu;
  shard_kv4_args a{};
  if (!p_keep || n != 8 || !integer(o[6], &device) || !integer(o[7], &stream) || !tensor(o[0], device, &cache) || !tensor(o[1], device, &table) ||
      !tensor(o[2], device, &lens) || !tensor(o[3], device, &rows) || !tensor(o[4], device, &counts) || !tensor(o[5], device, &cu, true))
    Py_RETURN_NONE;
  const int d = cache->dim() == 4 ? 1 : 0;
  if (table->dim() != 2 || !batch(a, cu ? INT32_MAX : table->size(0), *cache, *table, *lens, cu, d)) Py_RETURN_NONE;
  const int64_t L = d ? cache->size(0) : 1;
  if (L <= 0 || L > INT32_MAX || !indexes(*counts, a.batch) || rows->scalar_type() != at::kInt || rows->dim() != 2 ||
      rows->size(0) != a.batch || rows->size(1) <= 0 || rows->size(1) > INT32_MAX || (rows->stride(1) != 1 && rows->size(1) > 1))
    Py_RETURN_NONE;
  const int64_t width = rows->size(1), stride = a.batch > 1 ? rows->stride(0) : width;
  if (stride < width) Py_RETURN_NONE;
  int rc;
  {
    const Unlocked unlocked;
    rc = p_keep(&a, (int32_t)L, L > 1 ? cache->stride(0) : 0, (const int32_t*)rows->data_ptr(), stride, (int32_t)width,
                (const int32_t*)counts->data_ptr(), (void*)stream);
  }
  if (rc) Py_RETURN_NONE;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// verify_drafts(logits, tokens, parents, uniforms, cu_seqlens, draft_probs, temperature, max_new, max_depth, device, stream)
// -> path, counts, next_tokens
PyObject* verify(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t device, stream, width, depth = INT32_MAX;
  const at::Tensor *x, *tokens, *up, *u, *cu, *probs, *temps = nullptr;
  shard_verify_args a{};
  if (!p_verify || n != 11 || !integer(o[9], &device) || !integer(o[10], &stream) || !tensor(o[0], device, &x) || !tensor(o[1], device, &tokens) ||
      !tensor(o[2], device, &up) || !tensor(o[3], device, &u) || !tensor(o[4], device, &cu, true) || !tensor(o[5], device, &probs, true) ||
      (o[8] != Py_None && !integer(o[8], &depth)) || depth < 0)
    Py_RETURN_NONE;
  const auto type = x->scalar_type();
  const int code = type == at::kFloat ? SHARD_FP32 : half_code(*x);
  if (code < 0 || x->dim() != 2 || x->size(0) <= 0 || x->size(0) > INT32_MAX || x->size(1) <= 0 || x->stride(1) != 1 || x->stride(0) < 0)
    Py_RETURN_NONE;
  const int64_t T = x->size(0), V = x->size(1);
  if (tokens->scalar_type() != at::kLong || tokens->dim() != 1 || tokens->size(0) != T || !tokens->is_contiguous() || !indexes(*up, T) ||
      u->scalar_type() != at::kFloat || u->dim() != 2 || u->size(0) != T || u->size(1) != 2 || !u->is_contiguous() ||
      (cu && (cu->dim() != 1 || cu->size(0) < 2 || !indexes(*cu, cu->size(0)))) || !tree_width(o[7], T, &width))
    Py_RETURN_NONE;
  if (probs && (probs->scalar_type() != at::kFloat || probs->dim() != 2 || probs->size(0) != T || probs->size(1) != V ||
                probs->stride(1) != 1 || probs->stride(0) < 0))
    Py_RETURN_NONE;
  const int64_t B = cu ? cu->size(0) - 1 : T;
  if (B > INT32_MAX) Py_RETURN_NONE;
  if (PyFloat_CheckExact(o[6])) a.temperature = (float)PyFloat_AS_DOUBLE(o[6]);
  else if (!tensor(o[6], device, &temps) || temps->scalar_type() != at::kFloat || temps->dim() != 1 || temps->size(0) != B || !temps->is_contiguous())
    Py_RETURN_NONE;
  a.batch = (int32_t)B;
  a.n_tokens = (int32_t)T;
  a.vocab = V;
  a.logits = x->data_ptr();
  a.row_stride = x->stride(0);
  a.dtype = code;
  a.width = (int32_t)width;
  a.tokens = (const int64_t*)tokens->data_ptr();
  a.parents = (const int32_t*)up->data_ptr();
  a.uniforms = (const float*)u->data_ptr();
  a.cu_seqlens = cu ? (const int32_t*)cu->data_ptr() : nullptr;
  a.draft_probs = probs ? (const float*)probs->data_ptr() : nullptr;
  a.probs_stride = probs ? probs->stride(0) : 0;
  a.temperatures = temps ? (const float*)temps->data_ptr() : nullptr;
  a.max_depth = (int32_t)std::min<int64_t>(depth, INT32_MAX);
  const int64_t one[1] = {B}, two[2] = {B, width};
  at::Tensor path, counts, next;
  int rc;
  {
    const Unlocked unlocked;
    path = make(two, *x, at::kInt);
    counts = make(one, *x, at::kInt);
    next = make(one, *x, at::kLong);
    a.path = (int32_t*)path.data_ptr();
    a.counts = (int32_t*)counts.data_ptr();
    a.next = (int64_t*)next.data_ptr();
    const size_t need = p_verify_workspace(&a);
    const c10::DataPtr ws = scratch(need);
    rc = p_verify(&a, ws.get(), need, (void*)stream);
  }
  if (rc) Py_RETURN_NONE;
  return Py_BuildValue("NNN", THPVariable_Wrap(std::move(path)), THPVariable_Wrap(std::move(counts)), THPVariable_Wrap(std::move(next)));
  END_HANDLE_TH_ERRORS
}

// token_logprobs(logits, tokens, top, device, stream) -> logprob (or None), entropy, top_logprobs, top_ids
PyObject* logprobs(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t device, stream, top;
  const at::Tensor *x, *tok;
  if (n != 5 || !integer(o[3], &device) || !integer(o[4], &stream) || !integer(o[2], &top) || !tensor(o[0], device, &x) ||
      !tensor(o[1], device, &tok, true))
    Py_RETURN_NONE;
  const auto type = x->scalar_type();
  const int code = type == at::kFloat ? SHARD_FP32 : half_code(*x);
  if (code < 0 || x->dim() != 2 || x->size(0) <= 0 || x->size(1) <= 0 || x->stride(1) != 1 || top < 0 || top > 64 || top > x->size(1))
    Py_RETURN_NONE;
  const int64_t R = x->size(0), V = x->size(1);
  if (tok && (tok->scalar_type() != at::kLong || tok->dim() != 1 || tok->size(0) != R || !tok->is_contiguous())) Py_RETURN_NONE;
  const int64_t one[1] = {R}, two[2] = {R, top};
  at::Tensor entropy, top_lp, top_ids, lp;
  int rc;
  {
    const Unlocked unlocked;
    entropy = make(one, *x, at::kFloat);
    top_lp = make(two, *x, at::kFloat);
    top_ids = make(two, *x, at::kLong);
    if (tok) lp = make(one, *x, at::kFloat);
    const size_t need = p_logprobs_workspace(R, V, (int32_t)top);
    const c10::DataPtr ws = scratch(need);
    rc = p_logprobs(x->data_ptr(), code, R, V, x->stride(0), tok ? (const int64_t*)tok->data_ptr() : nullptr, (int32_t)top,
                    tok ? (float*)lp.data_ptr() : nullptr, (float*)entropy.data_ptr(), (float*)top_lp.data_ptr(),
                    (int64_t*)top_ids.data_ptr(), ws.get(), need, (void*)stream);
  }
  if (rc) Py_RETURN_NONE;
  PyObject* first = Py_None;
  if (tok) first = THPVariable_Wrap(std::move(lp));
  else Py_INCREF(Py_None);
  return Py_BuildValue("NNNN", first, THPVariable_Wrap(std::move(entropy)), THPVariable_Wrap(std::move(top_lp)),
                       THPVariable_Wrap(std::move(top_ids)));
  END_HANDLE_TH_ERRORS
}

// bind(path): the library's entry points; it is loaded already.  ImportError, and
// what was bound before stays, where it has not all of them or was built with
// another argument block than this file.
PyObject* bind(PyObject*, PyObject* path) {
  const char* p = PyUnicode_AsUTF8(path);
  if (!p) return nullptr;
  void* lib = dlopen(p, RTLD_NOW);
  if (!lib) return PyErr_Format(PyExc_ImportError, "%s", dlerror());
  const auto layout = (decltype(&shard_kv4_args_layout))dlsym(lib, "shard_kv4_args_layout");
  if (!layout || layout() != SHARD_KV4_ARGS_LAYOUT)
    return PyErr_Format(PyExc_ImportError, "%s was built with another shard_kv4_args", p);
  const char* const names[] = {"shard_kv4_append", "shard_kv4_read", "shard_kv4_attn_workspace", "shard_kv4_attn",
                               "shard_token_logprobs_workspace", "shard_token_logprobs"};
  void* f[6];
  for (int i = 0; i < 6; ++i)
    if (!(f[i] = dlsym(lib, names[i]))) return PyErr_Format(PyExc_ImportError, "%s misses %s", p, names[i]);
  p_append = (decltype(p_append))f[0];
  p_read = (decltype(p_read))f[1];
  p_attn_workspace = (decltype(p_attn_workspace))f[2];
  p_attn = (decltype(p_attn))f[3];
  p_logprobs_workspace = (decltype(p_logprobs_workspace))f[4];
  p_logprobs = (decltype(p_logprobs))f[5];
  // drafted tokens: all or none of them
  const char* const more[] = {"shard_kv4_append_at", "shard_kv4_tree_attn_workspace", "shard_kv4_tree_attn", "shard_kv4_keep",
                              "shard_draft_tree", "shard_verify_drafts_workspace", "shard_verify_drafts"};
  constexpr int N = sizeof(more) / sizeof(more[0]);
  void* g[N];
  const auto verify_size = (decltype(&shard_verify_args_size))dlsym(lib, "shard_verify_args_size");
  bool all = verify_size && verify_size() == sizeof(shard_verify_args);
  for (int i = 0; i < N; ++i) all = (g[i] = dlsym(lib, more[i])) && all;
  for (int i = 0; i < N && !all; ++i) g[i] = nullptr;
  p_append_at = (decltype(p_append_at))g[0];
  p_tree_workspace = (decltype(p_tree_workspace))g[1];
  p_tree_attn = (decltype(p_tree_attn))g[2];
  p_keep = (decltype(p_keep))g[3];
  p_tree = (decltype(p_tree))g[4];
  p_verify_workspace = (decltype(p_verify_workspace))g[5];
  p_verify = (decltype(p_verify))g[6];
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_O, nullptr},
    {"kv4_append", (PyCFunction)(void*)append, METH_FASTCALL, nullptr},
    {"kv4_read", (PyCFunction)(void*)read, METH_FASTCALL, nullptr},
    {"kv4_attn", (PyCFunction)(void*)attn, METH_FASTCALL, nullptr},
    {"kv4_tree_attn", (PyCFunction)(void*)attn, METH_FASTCALL, nullptr},
    {"draft_tree", (PyCFunction)(void*)tree, METH_FASTCALL, nullptr},
    {"kv4_keep", (PyCFunction)(void*)keep, METH_FASTCALL, nullptr},
    {"verify_drafts", (PyCFunction)(void*)verify, METH_FASTCALL, nullptr},
    {"token_logprobs", (PyCFunction)(void*)logprobs, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_dispatch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__dispatch(void) { return PyModule_Create(&module); }
