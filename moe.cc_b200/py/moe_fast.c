/*
 * moe_fast.c — the Python calls of a decode step (kv_plan, qk_norm_rope,
 * paged_attention, route of moe_cuda.py) as a CPython extension.
 *
 * These calls run kernels of 2 to 5 us. Checked and handed on by Python and
 * ctypes (moe_calls.py) they take the host 9 to 20 us, most of it for reading the
 * tensors' attributes and converting 20 arguments; from here they take 4 to 13.
 * Each tensor's type, device, shape and layout is checked before its pointer
 * goes on; a wrong one raises moe_cuda.MoeError, as an error of the library
 * does. torch is not linked: tensors are read through their Python attributes.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <limits.h>
#include <stdarg.h>

#include "../../include/moe_cuda.h"

static PyObject* g_error;                                  /* moe_cuda.MoeError */
static PyObject *s_shape, *s_stride, *s_dtype, *s_numel, *s_get_device, *s_is_contiguous, *s_data_ptr, *s_nbytes, *s_cuda_stream;
static PyObject *t_i32, *t_f32, *t_f16, *t_bf16;           /* torch's types, looked up with the first tensor */

static int refuse(int code, const char* fmt, ...) {
  va_list ap;
  PyErr_Clear();
  va_start(ap, fmt);
  PyObject* msg = PyUnicode_FromFormatV(fmt, ap);
  va_end(ap);
  if (!msg) return -1;
  PyObject* e = PyObject_CallFunction(g_error, "iO", code, msg);
  Py_DECREF(msg);
  if (!e) return -1;
  PyErr_SetObject(g_error, e);
  Py_DECREF(e);
  return -1;
}

static PyObject* done(int rc) {
  if (rc) { refuse(rc, "%s", moe_cuda_last_error()); return NULL; }
  Py_RETURN_NONE;
}

static int load_types(void) {
  if (t_bf16) return 0;
  PyObject* m = PyImport_ImportModule("torch");
  if (!m) return -1;
  t_i32 = PyObject_GetAttrString(m, "int32");
  t_f32 = PyObject_GetAttrString(m, "float32");
  t_f16 = PyObject_GetAttrString(m, "float16");
  t_bf16 = PyObject_GetAttrString(m, "bfloat16");
  Py_DECREF(m);
  return t_i32 && t_f32 && t_f16 && t_bf16 ? 0 : -1;
}

/* t.name() as an integer */
static int ask(PyObject* t, PyObject* name, long long* v) {
  PyObject* r = PyObject_CallMethodNoArgs(t, name);
  if (!r) return -1;
  *v = PyBool_Check(r) ? r == Py_True : (long long)PyLong_AsUnsignedLongLongMask(r);
  Py_DECREF(r);
  return PyErr_Occurred() ? -1 : 0;
}
/* t.dtype: the types live as long as torch does, so the reference is not kept */
static PyObject* type_of(PyObject* t) {
  PyObject* d = PyObject_GetAttr(t, s_dtype);
  if (d) Py_DECREF(d);
  else PyErr_Clear();
  return d;
}
static int elem_of(PyObject* dtype) {
  return dtype == t_f32 ? MOE_DTYPE_F32 : dtype == t_f16 ? MOE_DTYPE_F16 : dtype == t_bf16 ? MOE_DTYPE_BF16 : -1;
}

typedef struct {
  void* p;
  PyObject* dtype;
  long long dev, n[4], s[4];
  int nd;
} View;

static int tuple_of(PyObject* o, long long* v, int* n) {
  int ok = o && PyTuple_Check(o) && PyTuple_GET_SIZE(o) <= 4;
  if (ok) {
    *n = (int)PyTuple_GET_SIZE(o);
    for (int i = 0; i < *n; ++i) v[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(o, i));
  }
  Py_XDECREF(o);
  return ok && !PyErr_Occurred() ? 0 : -1;
}

/* shape, strides, type, device and address of a tensor of at most 4 dimensions */
static int view(PyObject* t, const char* what, View* v) {
  long long p;
  int ns;
  if (t == NULL || t == Py_None || tuple_of(PyObject_GetAttr(t, s_shape), v->n, &v->nd) ||
      tuple_of(PyObject_CallMethodNoArgs(t, s_stride), v->s, &ns) || ns != v->nd || ask(t, s_get_device, &v->dev) ||
      ask(t, s_data_ptr, &p) || !(v->dtype = type_of(t)))
    return refuse(MOE_ERR_INVALID, "%s: a tensor of at most 4 dimensions is wanted", what);
  v->p = (void*)(uintptr_t)p;
  return 0;
}

/* address of a contiguous tensor of n elements of one type on one device; None: NULL */
static int flat(PyObject* t, PyObject* dtype, long long n, long long dev, const char* what, void** p) {
  long long m, d, c, a;
  *p = NULL;
  if (t == NULL || t == Py_None) return 0;
  if (ask(t, s_numel, &m) || ask(t, s_get_device, &d) || ask(t, s_is_contiguous, &c) || ask(t, s_data_ptr, &a) ||
      m != n || (int)d != (int)dev || !c || type_of(t) != dtype)
    return refuse(MOE_ERR_INVALID, "%s: a contiguous tensor of %lld elements of %R on cuda:%d is wanted, got %R", what, n, dtype,
                  (int)dev, (PyObject*)Py_TYPE(t));
  *p = (void*)(uintptr_t)a;
  return 0;
}

/* [rows][heads][hd] whose rows may lie apart: address and row stride */
static int heads_of(PyObject* t, const char* what, long long rows, long long heads, long long hd, PyObject* dtype, long long dev,
                    void** p, long long* ld) {
  View v;
  if (view(t, what, &v)) return -1;
  if (v.nd != 3 || v.n[0] != rows || v.n[1] != heads || v.n[2] != hd || v.dev != dev || v.dtype != dtype ||
      (rows && ((v.s[2] != 1 && hd > 1) || (v.s[1] != hd && heads > 1))))
    return refuse(MOE_ERR_INVALID, "%s: [%lld][%lld][%lld] of %R on cuda:%d with contiguous rows is wanted", what, rows, heads, hd,
                  dtype, (int)dev);
  *p = v.p;
  *ld = rows > 1 ? v.s[0] : heads * hd;
  return 0;
}

/* two cache tensors [n_pages][page_size][n_kv][head_dim] of one type and layout */
static int cache_of(PyObject* k, PyObject* v, MoeKvCache* c, PyObject** dtype, long long* dev) {
  View a, b;
  if (load_types() || view(k, "k_cache", &a) || view(v, "v_cache", &b)) return -1;
  int same = a.nd == 4 && b.nd == 4 && a.dtype == b.dtype && a.dev == b.dev;
  for (int i = 0; same && i < 4; ++i) {
    if (a.n[i] == 1) a.s[i] = b.s[i] = i == 3 ? 1 : 0;     /* the stride of a dimension of one says nothing */
    same = a.n[i] == b.n[i] && a.s[i] == b.s[i] && a.n[i] <= INT_MAX;
  }
  const int dt = elem_of(a.dtype);
  if (!same || a.dev < 0 || dt < 0 || a.s[3] != 1)
    return refuse(MOE_ERR_INVALID, "kv cache: k and v of one type (float32, float16 or bfloat16) and layout, [n_pages][page_size]"
                  "[n_kv][head_dim], the last dimension contiguous, on a CUDA device");
  c->k = a.p; c->v = b.p; c->dtype = dt;
  c->n_pages = (int)a.n[0]; c->page_size = (int)a.n[1]; c->n_kv = (int)a.n[2]; c->head_dim = (int)a.n[3];
  c->page_stride = a.s[0]; c->token_stride = a.s[1]; c->head_stride = a.s[2];
  *dtype = a.dtype;
  *dev = a.dev;
  return 0;
}

static int integer(PyObject* o, const char* what, int* v) {
  *v = 0;
  const long long x = o ? PyLong_AsLongLong(o) : 0;
  if (!o || PyErr_Occurred() || x > INT_MAX || x < INT_MIN) return refuse(MOE_ERR_INVALID, "%s: a 32-bit integer is wanted", what);
  *v = (int)x;
  return 0;
}
static int real(PyObject* o, const char* what, double* v) {
  *v = o ? PyFloat_AsDouble(o) : 0;
  return !o || PyErr_Occurred() ? refuse(MOE_ERR_INVALID, "%s: a number is wanted", what) : 0;
}
/* None, a cudaStream_t as an integer, or an object with one in .cuda_stream */
static int stream_of(PyObject* o, void** s) {
  *s = NULL;
  if (o == NULL || o == Py_None) return 0;
  PyObject* n = PyLong_Check(o) ? Py_NewRef(o) : PyObject_GetAttr(o, s_cuda_stream);
  if (n) { *s = (void*)(uintptr_t)PyLong_AsUnsignedLongLong(n); Py_DECREF(n); }
  return PyErr_Occurred() ? refuse(MOE_ERR_INVALID, "stream: a CUDA stream is wanted") : 0;
}

/* Arguments by position and keyword into out[n]; the first `needed` have to be there. */
static int arguments(const char* who, PyObject* const* args, Py_ssize_t n_args, PyObject* kw, PyObject** names, int n, int needed,
                     PyObject** out) {
  if (n_args > n) { PyErr_Format(PyExc_TypeError, "%s() takes %d arguments", who, n); return -1; }
  for (int i = 0; i < n; ++i) out[i] = i < n_args ? args[i] : NULL;
  const Py_ssize_t n_kw = kw ? PyTuple_GET_SIZE(kw) : 0;
  for (Py_ssize_t k = 0; k < n_kw; ++k) {
    PyObject* name = PyTuple_GET_ITEM(kw, k);
    int i = 0;
    while (i < n && names[i] != name) ++i;                 /* interned, as keywords are */
    if (i == n)
      for (i = 0; i < n && PyUnicode_Compare(names[i], name) != 0; ++i) {}
    if (i == n || out[i]) { PyErr_Format(PyExc_TypeError, "%s() got %s argument '%U'", who, i == n ? "an unexpected" : "twice the", name); return -1; }
    out[i] = args[n_args + k];
  }
  for (int i = 0; i < needed; ++i)
    if (!out[i]) { PyErr_Format(PyExc_TypeError, "%s() needs '%U'", who, names[i]); return -1; }
  return 0;
}

#define MAX_ARGS 16
static PyObject* n_plan[MAX_ARGS];
static PyObject* n_rope[MAX_ARGS];
static PyObject* n_attn[MAX_ARGS];
static PyObject* n_route[MAX_ARGS];

static const char* const plan_names[] = {"past_len", "new_len", "page_size", "n_pages", "free_pages", "block_table", "row_seq",
                                         "row_pos", "row_slot", "kv_len", "free_head", "free_head_out", "status", "stream", NULL};
static PyObject* kv_plan(PyObject* self, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
  PyObject* a[14];
  View t;
  long long cap, n_free;
  int ps = 0, pages = 0;
  void *past, *fresh, *free_p, *head, *kv, *seq, *pos, *slot, *head_out, *status, *st;
  if (arguments("kv_plan", args, n, kw, n_plan, 14, 9, a) || load_types() || view(a[5], "block_table", &t)) return NULL;
  long long whole = t.nd == 2 ? t.n[0] * t.n[1] : -1;
  void* table;
  if (whole < 0 || t.dev < 0 || t.n[0] > INT_MAX || t.n[1] > INT_MAX) {
    refuse(MOE_ERR_INVALID, "block_table: [sequences][pages] on a CUDA device is wanted");
    return NULL;
  }
  if (ask(a[6], s_numel, &cap) || ask(a[4], s_numel, &n_free)) {
    refuse(MOE_ERR_INVALID, "row_seq, free_pages: tensors are wanted");
    return NULL;
  }
  if (flat(a[5], t_i32, whole, t.dev, "block_table", &table) || integer(a[2], "page_size", &ps) || integer(a[3], "n_pages", &pages) || flat(a[0], t_i32, t.n[0], t.dev, "past_len", &past) ||
      flat(a[1], t_i32, t.n[0], t.dev, "new_len", &fresh) || flat(a[4], t_i32, n_free, t.dev, "free_pages", &free_p) ||
      flat(a[6], t_i32, cap, t.dev, "row_seq", &seq) || flat(a[7], t_i32, cap, t.dev, "row_pos", &pos) ||
      flat(a[8], t_i32, cap, t.dev, "row_slot", &slot) || flat(a[9], t_i32, t.n[0], t.dev, "kv_len", &kv) ||
      flat(a[10], t_i32, 1, t.dev, "free_head", &head) || flat(a[11], t_i32, 1, t.dev, "free_head_out", &head_out) ||
      flat(a[12], t_i32, 3, t.dev, "status", &status) || stream_of(a[13], &st))
    return NULL;
  if (cap > INT_MAX || n_free > INT_MAX) { refuse(MOE_ERR_UNSUPPORTED, "kv_plan: more than 2^31 - 1 rows or free pages"); return NULL; }
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = moe_kv_plan_dev(past, fresh, (int)t.n[0], ps, pages, free_p, (int)n_free, head, table, (int)t.n[1], kv, seq, pos, slot,
                       (int)cap, head_out, status, st);
  Py_END_ALLOW_THREADS
  return done(rc);
}

static const char* const rope_names[] = {"q", "k", "v", "k_cache", "v_cache", "row_pos", "row_slot", "q_out", "rope", "q_norm",
                                         "k_norm", "eps", "stream", NULL};
static PyObject* qk_norm_rope(PyObject* self, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
  PyObject *a[13], *ct;
  MoeKvCache c;
  View x, r;
  long long dev, ldq = 0, ldo = 0, ldk = 0, ldv = 0, heads = 0, n_rope_rows = 0, rot = 0;
  void *q = NULL, *o = NULL, *k = NULL, *v = NULL, *pos, *slot, *qn, *kn, *rp = NULL, *st;
  double eps = 1e-6;
  if (arguments("qk_norm_rope", args, n, kw, n_rope, 13, 8, a) || cache_of(a[3], a[4], &c, &ct, &dev)) return NULL;
  const int hd = c.head_dim, with_q = a[0] != Py_None, append = a[6] != Py_None;
  if (view(with_q ? a[0] : a[1], with_q ? "q" : "k", &x)) return NULL;
  const int dt = elem_of(x.dtype);
  if (dt < 0 || x.nd != 3 || x.n[0] > INT_MAX || x.n[1] > INT_MAX) {
    refuse(MOE_ERR_INVALID, "q, k: [rows][heads][head_dim] of float32, float16 or bfloat16 is wanted");
    return NULL;
  }
  const long long rows = x.n[0];
  if (with_q) {
    heads = x.n[1];
    if (heads_of(a[0], "q", rows, heads, hd, x.dtype, dev, &q, &ldq) || heads_of(a[7], "q_out", rows, heads, hd, ct, dev, &o, &ldo))
      return NULL;
  }
  if (append && (heads_of(a[1], "k", rows, c.n_kv, hd, x.dtype, dev, &k, &ldk) ||
                 heads_of(a[2], "v", rows, c.n_kv, hd, x.dtype, dev, &v, &ldv)))
    return NULL;
  if (a[8] && a[8] != Py_None) {
    if (view(a[8], "rope", &r)) return NULL;
    if (r.nd != 2 || r.n[0] > INT_MAX || r.n[1] > INT_MAX) { refuse(MOE_ERR_INVALID, "rope: [positions][rot_dim] is wanted"); return NULL; }
    n_rope_rows = r.n[0];
    rot = r.n[1];
  }
  if (flat(a[5], t_i32, rows, dev, "row_pos", &pos) || flat(a[6], t_i32, rows, dev, "row_slot", &slot) ||
      flat(a[8], t_f32, n_rope_rows * rot, dev, "rope", &rp) || flat(a[9], t_f32, hd, dev, "q_norm", &qn) ||
      flat(a[10], t_f32, hd, dev, "k_norm", &kn) || (a[11] && real(a[11], "eps", &eps)) || stream_of(a[12], &st))
    return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = moe_qk_norm_rope_dev(q, ldq, k, ldk, v, ldv, dt, (int)rows, (int)heads, qn, kn, (float)eps, rp, (int)rot, (int)n_rope_rows,
                            pos, slot, o, ldo, &c, st);
  Py_END_ALLOW_THREADS
  return done(rc);
}

static const char* const attn_names[] = {"q", "k_cache", "v_cache", "block_table", "row_pos", "out", "workspace", "max_kv", "scale",
                                         "lse", "row_seq", "stream", NULL};
static PyObject* paged_attention(PyObject* self, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
  PyObject *a[12], *ct;
  MoeKvCache c;
  View x, t;
  long long dev, ldq, ldo, ws_bytes = 0, ws_dev, ws_flat, ws_p;
  void *q, *o, *table, *pos, *lse, *seq, *ws = NULL, *st;
  int max_kv = 0;
  double scale = 0;
  if (arguments("paged_attention", args, n, kw, n_attn, 12, 9, a) || cache_of(a[1], a[2], &c, &ct, &dev) ||
      view(a[0], "q", &x) || view(a[3], "block_table", &t))
    return NULL;
  if (x.nd != 3 || t.nd != 2 || x.n[0] > INT_MAX || x.n[1] > INT_MAX || t.n[0] > INT_MAX || t.n[1] > INT_MAX) {
    refuse(MOE_ERR_INVALID, "q: [rows][heads][head_dim], block_table: [sequences][pages] are wanted");
    return NULL;
  }
  const long long rows = x.n[0], heads = x.n[1];
  if (heads_of(a[0], "q", rows, heads, c.head_dim, ct, dev, &q, &ldq) ||
      heads_of(a[5], "out", rows, heads, c.head_dim, ct, dev, &o, &ldo) ||
      flat(a[3], t_i32, t.n[0] * t.n[1], dev, "block_table", &table) || flat(a[4], t_i32, rows, dev, "row_pos", &pos) ||
      flat(a[9], t_f32, rows * heads, dev, "lse", &lse) || flat(a[10], t_i32, rows, dev, "row_seq", &seq) ||
      integer(a[7], "max_kv", &max_kv) || real(a[8], "scale", &scale) || stream_of(a[11], &st))
    return NULL;
  if (a[6] != Py_None) {
    PyObject* nb = PyObject_GetAttr(a[6], s_nbytes);
    if (nb) { ws_bytes = PyLong_AsLongLong(nb); Py_DECREF(nb); }
    if (PyErr_Occurred() || ask(a[6], s_get_device, &ws_dev) || ask(a[6], s_is_contiguous, &ws_flat) || ask(a[6], s_data_ptr, &ws_p) ||
        (int)ws_dev != (int)dev || !ws_flat) {
      refuse(MOE_ERR_INVALID, "workspace: a contiguous tensor on cuda:%d is wanted", (int)dev);
      return NULL;
    }
    ws = (void*)(uintptr_t)ws_p;
  }
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = moe_paged_attention_dev(q, ldq, &c, table, (int)t.n[0], (int)t.n[1], seq, pos, (int)rows, (int)heads, max_kv, (float)scale, o,
                               ldo, lse, ws, (size_t)ws_bytes, st);
  Py_END_ALLOW_THREADS
  return done(rc);
}

static const char* const route_names[] = {"logits", "topk_idx", "topk_p", "bias", "score", "groups", "keep_groups", "group_top",
                                          "renorm", "scale", "stream", NULL};
static PyObject* route(PyObject* self, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
  PyObject* a[11];
  View x, i;
  void *idx, *p, *bias, *st;
  int score = MOE_ROUTE_SOFTMAX, groups = 1, keep = 1, top = 1, renorm = 1;
  double scale = 1.0;
  if (arguments("route", args, n, kw, n_route, 11, 3, a) || load_types() || view(a[0], "logits", &x) || view(a[1], "topk_idx", &i))
    return NULL;
  const int dt = elem_of(x.dtype);
  if (dt < 0 || x.nd != 2 || i.nd != 2 || x.dev < 0 || x.n[0] > INT_MAX || x.n[1] > INT_MAX || i.n[1] > INT_MAX ||
      (x.n[0] && x.n[1] > 1 && x.s[1] != 1)) {
    refuse(MOE_ERR_INVALID, "logits: [rows][experts] of float32, float16 or bfloat16 with contiguous experts on a CUDA device, "
           "topk_idx: [rows][top_k] are wanted");
    return NULL;
  }
  if (a[4]) {
    if (PyUnicode_Check(a[4]) && PyUnicode_CompareWithASCIIString(a[4], "sigmoid") == 0) score = MOE_ROUTE_SIGMOID;
    else if (!PyUnicode_Check(a[4]) || PyUnicode_CompareWithASCIIString(a[4], "softmax") != 0) {
      refuse(MOE_ERR_INVALID, "score: 'softmax' or 'sigmoid' is wanted");
      return NULL;
    }
  }
  const long long rows = x.n[0], k = i.n[1];
  if (flat(a[1], t_i32, rows * k, x.dev, "topk_idx", &idx) || flat(a[2], t_f32, rows * k, x.dev, "topk_p", &p) ||
      flat(a[3], t_f32, x.n[1], x.dev, "bias", &bias) || (a[5] && integer(a[5], "groups", &groups)) ||
      (a[6] && integer(a[6], "keep_groups", &keep)) || (a[7] && integer(a[7], "group_top", &top)) ||
      (a[8] && (renorm = PyObject_IsTrue(a[8])) < 0) || (a[9] && real(a[9], "scale", &scale)) || stream_of(a[10], &st))
    return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = moe_route_dev(x.p, rows > 1 ? x.s[0] : x.n[1], dt, (int)rows, (int)x.n[1], bias, score, groups, keep, top, (int)k, renorm, scale,
                     idx, p, st);
  Py_END_ALLOW_THREADS
  return done(rc);
}

static PyObject* set_error(PyObject* self, PyObject* cls) {
  Py_XSETREF(g_error, Py_NewRef(cls));
  Py_RETURN_NONE;
}

#define FAST (PyCFunction)(void (*)(void))
static PyMethodDef methods[] = {
    {"kv_plan", FAST kv_plan, METH_FASTCALL | METH_KEYWORDS,
     "kv_plan(past_len, new_len, page_size, n_pages, free_pages, block_table, row_seq, row_pos, row_slot, kv_len=None,\n"
     "        free_head=None, free_head_out=None, status=None, stream=None)\n\n"
     "moe_kv_plan_dev on int32 tensors; past_len may be None (nothing held yet). block_table [sequences][pages]; the three\n"
     "row tensors of one length; free_head, free_head_out of one element, status of three."},
    {"qk_norm_rope", FAST qk_norm_rope, METH_FASTCALL | METH_KEYWORDS,
     "qk_norm_rope(q, k, v, k_cache, v_cache, row_pos, row_slot, q_out, rope=None, q_norm=None, k_norm=None, eps=1e-6,\n"
     "             stream=None)\n\n"
     "moe_qk_norm_rope_dev. q [rows][n_q][head_dim] (None: keys and values only), k, v [rows][n_kv][head_dim], rows of one\n"
     "stride each; rope [positions][rot_dim] fp32, the cosines then the sines; row_slot None: queries only (k, v are then\n"
     "not read and may be None)."},
    {"paged_attention", FAST paged_attention, METH_FASTCALL | METH_KEYWORDS,
     "paged_attention(q, k_cache, v_cache, block_table, row_pos, out, workspace, max_kv, scale, lse=None, row_seq=None,\n"
     "                stream=None)\n\n"
     "moe_paged_attention_dev. q, out [rows][n_q][head_dim]; workspace: a contiguous tensor of any type (None where none is\n"
     "needed)."},
    {"route", FAST route, METH_FASTCALL | METH_KEYWORDS,
     "route(logits, topk_idx, topk_p, bias=None, score='softmax', groups=1, keep_groups=1, group_top=1, renorm=True,\n"
     "      scale=1.0, stream=None)\n\n"
     "moe_route_dev: topk_idx (int32) and topk_p (fp32) [rows][top_k] of logits [rows][experts] (rows may lie apart);\n"
     "score 'softmax' or 'sigmoid'."},
    {"_set_error", set_error, METH_O, "The exception that refusals and errors raise: called with a code and a message."},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_moe_fast", "Calls of a decode step (see moe_cuda.py).", -1, methods};

static int intern(const char* const* from, PyObject** to) {
  for (int i = 0; from[i]; ++i)
    if (!(to[i] = PyUnicode_InternFromString(from[i]))) return -1;
  return 0;
}

PyMODINIT_FUNC PyInit__moe_fast(void) {
  static const char* const attrs[] = {"shape", "stride", "dtype", "numel", "get_device", "is_contiguous", "data_ptr", "nbytes",
                                      "cuda_stream", NULL};
  PyObject* v[9];
  if (intern(attrs, v) || intern(plan_names, n_plan) || intern(rope_names, n_rope) || intern(attn_names, n_attn) ||
      intern(route_names, n_route))
    return NULL;
  s_shape = v[0]; s_stride = v[1]; s_dtype = v[2]; s_numel = v[3]; s_get_device = v[4]; s_is_contiguous = v[5];
  s_data_ptr = v[6]; s_nbytes = v[7]; s_cuda_stream = v[8];
  g_error = Py_NewRef(PyExc_RuntimeError);
  return PyModule_Create(&module);
}
