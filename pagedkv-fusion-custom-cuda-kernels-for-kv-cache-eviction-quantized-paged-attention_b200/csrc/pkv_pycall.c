/* Direct CPython calls into the C ABI for the eviction latency path and the
 * prompt, shared-prefix and growing-cache operators.
 *
 * The eviction decision (score 16K blocks, select the k lowest) takes
 * ~13 us on the GPU, so the host cost of reaching the launch matters: a
 * ctypes call with 15 converted arguments costs ~2.2 us, this module's
 * METH_FASTCALL functions ~0.2 us.  Each function takes the C ABI
 * entry point's arguments in order -- device pointers and the stream as
 * Python ints (None for a null pointer), sizes as ints, weights as floats
 * -- and returns its status code; pagedkv_fusion._C checks the tensors and
 * raises on a nonzero status exactly as on its ctypes path.  Built by
 * build.py with the host C compiler against this interpreter's headers and
 * linked to libpagedkv_sm100.so beside it.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

#include "pagedkv_fusion.h"

static int as_ptr(PyObject* o, void** out) {
  if (o == Py_None) {
    *out = NULL;
    return 0;
  }
  *out = PyLong_AsVoidPtr(o);
  return (*out == NULL && PyErr_Occurred()) ? -1 : 0;
}

static int as_i64(PyObject* o, int64_t* out) {
  *out = (int64_t)PyLong_AsLongLong(o);
  return (*out == -1 && PyErr_Occurred()) ? -1 : 0;
}

static int as_i32(PyObject* o, int32_t* out) {
  int64_t v;
  if (as_i64(o, &v)) return -1;
  if (v < INT32_MIN || v > INT32_MAX) {
    PyErr_SetString(PyExc_OverflowError, "size does not fit in 32 bits");
    return -1;
  }
  *out = (int32_t)v;
  return 0;
}

static int as_f32(PyObject* o, float* out) {
  const double d = PyFloat_AsDouble(o);
  if (d == -1.0 && PyErr_Occurred()) return -1;
  *out = (float)d;
  return 0;
}

static int nargs_ok(Py_ssize_t got, Py_ssize_t want, const char* name) {
  if (got == want) return 1;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (%zd given)", name, want, got);
  return 0;
}

/* eviction_scores(rec, freq, attn, valid, out, num_blocks, block_size,
 *                 w_recency, w_frequency, w_attention, stream) */
static PyObject* py_eviction_scores(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  void *rec, *freq, *attn, *valid, *out, *stream;
  int64_t nb, bs;
  float wr, wf, wa;
  (void)self;
  if (!nargs_ok(n, 11, "eviction_scores")) return NULL;
  if (as_ptr(a[0], &rec) || as_ptr(a[1], &freq) || as_ptr(a[2], &attn) || as_ptr(a[3], &valid) ||
      as_ptr(a[4], &out) || as_i64(a[5], &nb) || as_i64(a[6], &bs) || as_f32(a[7], &wr) ||
      as_f32(a[8], &wf) || as_f32(a[9], &wa) || as_ptr(a[10], &stream))
    return NULL;
  return PyLong_FromLong(pkv_eviction_scores((const float*)rec, (const float*)freq,
                                             (const float*)attn, (const uint8_t*)valid,
                                             (float*)out, nb, (int32_t)bs, wr, wf, wa, stream));
}

/* eviction_select(scores, num_blocks, k, out, workspace, workspace_bytes, stream) */
static PyObject* py_eviction_select(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  void *scores, *out, *ws, *stream;
  int64_t nb, k, wsb;
  (void)self;
  if (!nargs_ok(n, 7, "eviction_select")) return NULL;
  if (as_ptr(a[0], &scores) || as_i64(a[1], &nb) || as_i64(a[2], &k) || as_ptr(a[3], &out) ||
      as_ptr(a[4], &ws) || as_i64(a[5], &wsb) || as_ptr(a[6], &stream))
    return NULL;
  return PyLong_FromLong(pkv_eviction_select((const float*)scores, nb, k, (int64_t*)out, ws,
                                             (size_t)wsb, stream));
}

/* eviction_scores_select(rec, freq, attn, valid, scores, num_blocks,
 *   block_size, w_recency, w_frequency, w_attention, k, out, workspace,
 *   workspace_bytes, stream) */
static PyObject* py_eviction_scores_select(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  void *rec, *freq, *attn, *valid, *scores, *out, *ws, *stream;
  int64_t nb, bs, k, wsb;
  float wr, wf, wa;
  (void)self;
  if (!nargs_ok(n, 15, "eviction_scores_select")) return NULL;
  if (as_ptr(a[0], &rec) || as_ptr(a[1], &freq) || as_ptr(a[2], &attn) || as_ptr(a[3], &valid) ||
      as_ptr(a[4], &scores) || as_i64(a[5], &nb) || as_i64(a[6], &bs) || as_f32(a[7], &wr) ||
      as_f32(a[8], &wf) || as_f32(a[9], &wa) || as_i64(a[10], &k) || as_ptr(a[11], &out) ||
      as_ptr(a[12], &ws) || as_i64(a[13], &wsb) || as_ptr(a[14], &stream))
    return NULL;
  return PyLong_FromLong(pkv_eviction_scores_select(
      (const float*)rec, (const float*)freq, (const float*)attn, (const uint8_t*)valid,
      (float*)scores, nb, (int32_t)bs, wr, wf, wa, k, (int64_t*)out, ws, (size_t)wsb, stream));
}

/* The C arguments of the functions below are read in order from a[0 ..]. */
#define PTR(i, v) as_ptr(a[i], &v)
#define I32(i, v) as_i32(a[i], &v)
#define I64(i, v) as_i64(a[i], &v)
#define F32(i, v) as_f32(a[i], &v)

/* The arguments of pkv_qk_norm_rope. */
static PyObject* py_qk_norm_rope(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  void *q, *k, *qo, *ko, *pos, *table, *qw, *kw, *stream;
  int32_t dtype, wf, heads, kv, dim, rot, inter;
  int64_t tokens, rows, qt, qh, kt, kh;
  float eps;
  (void)self;
  if (!nargs_ok(n, 23, "qk_norm_rope")) return NULL;
  if (PTR(0, q) || PTR(1, k) || I32(2, dtype) || PTR(3, qo) || PTR(4, ko) || PTR(5, pos) ||
      PTR(6, table) || PTR(7, qw) || PTR(8, kw) || I32(9, wf) || F32(10, eps) || I64(11, tokens) ||
      I32(12, heads) || I32(13, kv) || I32(14, dim) || I32(15, rot) || I64(16, rows) ||
      I32(17, inter) || I64(18, qt) || I64(19, qh) || I64(20, kt) || I64(21, kh) ||
      PTR(22, stream))
    return NULL;
  return PyLong_FromLong(pkv_qk_norm_rope(q, k, dtype, qo, ko, pos, table, qw, kw, wf, eps, tokens,
                                          heads, kv, dim, rot, rows, inter, qt, qh, kt, kh,
                                          stream));
}

/* The arguments of pkv_append_kv. */
static PyObject* py_append_kv(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  void *key, *value, *cache, *scales, *slots, *pos, *table, *ws, *stream;
  int32_t dtype, bs, kv, dim, rot, inter;
  int64_t tokens, blocks, rows, kt, kh, vt, vh, wsb;
  (void)self;
  if (!nargs_ok(n, 23, "append_kv")) return NULL;
  if (PTR(0, key) || PTR(1, value) || I32(2, dtype) || PTR(3, cache) || PTR(4, scales) ||
      PTR(5, slots) || PTR(6, pos) || PTR(7, table) || I64(8, tokens) || I64(9, blocks) ||
      I32(10, bs) || I32(11, kv) || I32(12, dim) || I32(13, rot) || I64(14, rows) ||
      I32(15, inter) || I64(16, kt) || I64(17, kh) || I64(18, vt) || I64(19, vh) || PTR(20, ws) ||
      I64(21, wsb) || PTR(22, stream))
    return NULL;
  return PyLong_FromLong(pkv_append_kv(key, value, dtype, cache, scales, slots, pos, table, tokens,
                                       blocks, bs, kv, dim, rot, rows, inter, kt, kh, vt, vh, ws,
                                       (size_t)wsb, stream));
}

/* The arguments of pkv_prefill_attention_ws. */
static PyObject* py_prefill_attention(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  void *q, *k, *v, *out, *lse, *cq, *ck, *ws, *stream;
  int32_t dtype, seqs, heads, kv, dim, causal;
  int64_t tq, tk, qt, qh, kt, kh, vt, vh, wsb;
  float scale;
  (void)self;
  if (!nargs_ok(n, 25, "prefill_attention")) return NULL;
  if (PTR(0, q) || PTR(1, k) || PTR(2, v) || I32(3, dtype) || PTR(4, out) || PTR(5, lse) ||
      PTR(6, cq) || PTR(7, ck) || I32(8, seqs) || I64(9, tq) || I64(10, tk) || I32(11, heads) ||
      I32(12, kv) || I32(13, dim) || I64(14, qt) || I64(15, qh) || I64(16, kt) || I64(17, kh) ||
      I64(18, vt) || I64(19, vh) || F32(20, scale) || I32(21, causal) || PTR(22, ws) ||
      I64(23, wsb) || PTR(24, stream))
    return NULL;
  return PyLong_FromLong(pkv_prefill_attention_ws(q, k, v, dtype, out, lse, cq, ck, seqs, tq, tk,
                                                  heads, kv, dim, qt, qh, kt, kh, vt, vh, scale,
                                                  causal, ws, (size_t)wsb, stream));
}

/* The arguments of pkv_shared_prefix_attention. */
static PyObject* py_shared_prefix_attention(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  void *q, *kc, *ks, *vc, *vs, *pt, *pl, *bt, *sl, *out, *ws, *stream;
  int32_t seqs, heads, kv, dim, bs, width, own;
  int64_t blocks, wsb;
  float scale;
  (void)self;
  if (!nargs_ok(n, 22, "shared_prefix_attention")) return NULL;
  if (PTR(0, q) || PTR(1, kc) || PTR(2, ks) || PTR(3, vc) || PTR(4, vs) || PTR(5, pt) ||
      PTR(6, pl) || PTR(7, bt) || PTR(8, sl) || PTR(9, out) || I32(10, seqs) || I32(11, heads) ||
      I32(12, kv) || I32(13, dim) || I32(14, bs) || I64(15, blocks) || I32(16, width) ||
      I32(17, own) || F32(18, scale) || PTR(19, ws) || I64(20, wsb) || PTR(21, stream))
    return NULL;
  return PyLong_FromLong(pkv_shared_prefix_attention(q, kc, ks, vc, vs, pt, pl, bt, sl, out, seqs,
                                                     heads, kv, dim, bs, blocks, width, own, scale,
                                                     ws, (size_t)wsb, stream));
}

/* The arguments of pkv_chunk_attention. */
static PyObject* py_chunk_attention(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  void *q, *kc, *ks, *vc, *vs, *bt, *sl, *cu, *out, *lse, *ws, *stream;
  int32_t dtype, seqs, heads, kv, dim, bs, width;
  int64_t tq, blocks, qt, qh, wsb;
  float scale;
  (void)self;
  if (!nargs_ok(n, 25, "chunk_attention")) return NULL;
  if (PTR(0, q) || I32(1, dtype) || PTR(2, kc) || PTR(3, ks) || PTR(4, vc) || PTR(5, vs) ||
      PTR(6, bt) || PTR(7, sl) || PTR(8, cu) || PTR(9, out) || PTR(10, lse) || I64(11, tq) ||
      I32(12, seqs) || I32(13, heads) || I32(14, kv) || I32(15, dim) || I32(16, bs) ||
      I64(17, blocks) || I32(18, width) || I64(19, qt) || I64(20, qh) || F32(21, scale) ||
      PTR(22, ws) || I64(23, wsb) || PTR(24, stream))
    return NULL;
  return PyLong_FromLong(pkv_chunk_attention(q, dtype, kc, ks, vc, vs, bt, sl, cu, out, lse, tq,
                                             seqs, heads, kv, dim, bs, blocks, width, qt, qh,
                                             scale, ws, (size_t)wsb, stream));
}

/* The arguments of pkv_accumulate_attention. */
static PyObject* py_accumulate_attention(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  void *w, *q, *kc, *ks, *bt, *sl, *cu, *lse, *ws, *stream;
  int32_t dtype, seqs, heads, kv, dim, bs, width;
  int64_t tq, blocks, qt, qh, wsb;
  float scale;
  (void)self;
  if (!nargs_ok(n, 23, "accumulate_attention")) return NULL;
  if (PTR(0, w) || PTR(1, q) || I32(2, dtype) || PTR(3, kc) || PTR(4, ks) || PTR(5, bt) ||
      PTR(6, sl) || PTR(7, cu) || PTR(8, lse) || I64(9, tq) || I32(10, seqs) || I32(11, heads) ||
      I32(12, kv) || I32(13, dim) || I32(14, bs) || I64(15, blocks) || I32(16, width) ||
      I64(17, qt) || I64(18, qh) || F32(19, scale) || PTR(20, ws) || I64(21, wsb) ||
      PTR(22, stream))
    return NULL;
  return PyLong_FromLong(pkv_accumulate_attention(w, q, dtype, kc, ks, bt, sl, cu, lse, tq, seqs,
                                                  heads, kv, dim, bs, blocks, width, qt, qh, scale,
                                                  ws, (size_t)wsb, stream));
}

/* The arguments of pkv_evict_tokens. */
static PyObject* py_evict_tokens(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  void *cache, *scales, *w, *bt, *sl, *lens, *kept, *stream;
  int32_t seqs, bs, kv, dim, width, keep, sinks, recent;
  int64_t blocks;
  (void)self;
  if (!nargs_ok(n, 17, "evict_tokens")) return NULL;
  if (PTR(0, cache) || PTR(1, scales) || PTR(2, w) || PTR(3, bt) || PTR(4, sl) || PTR(5, lens) ||
      PTR(6, kept) || I32(7, seqs) || I64(8, blocks) || I32(9, bs) || I32(10, kv) || I32(11, dim) ||
      I32(12, width) || I32(13, keep) || I32(14, sinks) || I32(15, recent) || PTR(16, stream))
    return NULL;
  return PyLong_FromLong(pkv_evict_tokens(cache, scales, w, bt, sl, lens, kept, seqs, blocks, bs,
                                          kv, dim, width, keep, sinks, recent, stream));
}

static PyMethodDef kMethods[] = {
    {"eviction_scores", (PyCFunction)(void (*)(void))py_eviction_scores, METH_FASTCALL,
     "pkv_eviction_scores; returns the status code"},
    {"eviction_select", (PyCFunction)(void (*)(void))py_eviction_select, METH_FASTCALL,
     "pkv_eviction_select; returns the status code"},
    {"eviction_scores_select", (PyCFunction)(void (*)(void))py_eviction_scores_select,
     METH_FASTCALL, "pkv_eviction_scores_select; returns the status code"},
    {"qk_norm_rope", (PyCFunction)(void (*)(void))py_qk_norm_rope, METH_FASTCALL,
     "pkv_qk_norm_rope; returns the status code"},
    {"append_kv", (PyCFunction)(void (*)(void))py_append_kv, METH_FASTCALL,
     "pkv_append_kv; returns the status code"},
    {"prefill_attention", (PyCFunction)(void (*)(void))py_prefill_attention, METH_FASTCALL,
     "pkv_prefill_attention_ws; returns the status code"},
    {"shared_prefix_attention", (PyCFunction)(void (*)(void))py_shared_prefix_attention,
     METH_FASTCALL, "pkv_shared_prefix_attention; returns the status code"},
    {"chunk_attention", (PyCFunction)(void (*)(void))py_chunk_attention, METH_FASTCALL,
     "pkv_chunk_attention; returns the status code"},
    {"accumulate_attention", (PyCFunction)(void (*)(void))py_accumulate_attention, METH_FASTCALL,
     "pkv_accumulate_attention; returns the status code"},
    {"evict_tokens", (PyCFunction)(void (*)(void))py_evict_tokens, METH_FASTCALL,
     "pkv_evict_tokens; returns the status code"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_pkv_pycall",
                                     "Direct calls into libpagedkv_sm100.so", -1, kMethods};

PyMODINIT_FUNC PyInit__pkv_pycall(void) { return PyModule_Create(&kModule); }
