/* _fgc: the hot methods of the Python Tensor (ferrograd_amd.Tensor) as a
 * CPython extension type over the C-ABI in include/ferrograd.h.
 *
 * Building a lazy graph from Python calls one C-ABI function per op
 * (tensor.rs:442-778); through ctypes each call costs about 1.5-2 us of
 * argument conversion and wrapper objects on top of the op itself, which
 * made a Python-driven realise of ((x*0.5)+1).relu().sum(1) host-bound. Here
 * each op is one C call from the interpreter: the handle lives in the object,
 * results are new objects of the caller's type, and errors raise the
 * package's FerrogradError with fg_last_error()'s message. Everything else
 * (construction from host data, reads, backward) stays in the Python class,
 * which subclasses this type.
 *
 * realize_many and gradient let other Python threads run meanwhile, as the
 * calls through ctypes do: they compile kernels, wait for devices and walk
 * whole graphs. Tensors that another thread drops then, by collecting garbage for
 * one, wait for the call's end: the library takes one call at a time. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <limits.h>
#include <math.h>

#include "ferrograd.h"

static PyObject* g_error_class = NULL; /* FerrogradError, registered by the package */

typedef struct {
  PyObject_HEAD fg_tensor* h;
  PyObject* weakrefs;
} TensorObject;

static PyObject* raise_last(void) {
  PyErr_SetString(g_error_class ? g_error_class : PyExc_RuntimeError, fg_last_error());
  return NULL;
}

/* A new object of `tp` owning handle `h`. */
static PyObject* wrap(PyTypeObject* tp, fg_tensor* h) {
  TensorObject* o = (TensorObject*)tp->tp_alloc(tp, 0);
  if (!o) {
    fg_tensor_free(h);
    return NULL;
  }
  o->h = h;
  return (PyObject*)o;
}

static int check_tensor(PyObject* o, TensorObject** out);

/* Every op needs a handle: Tensor() without one is an empty shell. */
static int has_handle(TensorObject* t) {
  if (t->h) return 1;
  PyErr_SetString(g_error_class ? g_error_class : PyExc_RuntimeError, "tensor has no handle");
  return 0;
}

static void t_dealloc(TensorObject* self) {
  if (self->weakrefs) PyObject_ClearWeakRefs((PyObject*)self);
  if (self->h) fg_tensor_free(self->h);
  self->h = NULL;
  Py_TYPE(self)->tp_free((PyObject*)self);
}

/* Tensor(handle): adopt a handle the C-ABI returned (an int or None). */
static int t_init(TensorObject* self, PyObject* args, PyObject* kw) {
  PyObject* hv = Py_None;
  if (!PyArg_ParseTuple(args, "|O", &hv)) return -1;
  if (self->h) {
    fg_tensor_free(self->h);
    self->h = NULL;
  }
  if (hv == Py_None) return 0;
  void* p = PyLong_AsVoidPtr(hv);
  if (!p && PyErr_Occurred()) return -1;
  self->h = (fg_tensor*)p;
  return 0;
}

static PyObject* t_get_h(TensorObject* self, void* closure) {
  (void)closure;
  if (!self->h) Py_RETURN_NONE;
  return PyLong_FromVoidPtr(self->h);
}

static PyObject* unary(TensorObject* self, int op) {
  if (!has_handle(self)) return NULL;
  fg_tensor* out = NULL;
  if (fg_tensor_unary(self->h, op, &out)) return raise_last();
  return wrap(Py_TYPE(self), out);
}

static PyObject* binary(TensorObject* self, PyObject* other, int op) {
  TensorObject* o;
  if (check_tensor(other, &o) || !has_handle(self) || !has_handle(o)) return NULL;
  fg_tensor* out = NULL;
  if (fg_tensor_binary(self->h, o->h, op, &out)) return raise_last();
  return wrap(Py_TYPE(self), out);
}

/* A sequence of ints as int64 (at most 16: tensors here have few dims). */
static int int64s(PyObject* seq, int64_t* buf, int* n) {
  PyObject* f = PySequence_Fast(seq, "expected a sequence of ints");
  if (!f) return -1;
  Py_ssize_t len = PySequence_Fast_GET_SIZE(f);
  if (len > 16) {
    Py_DECREF(f);
    PyErr_SetString(PyExc_ValueError, "at most 16 dimensions");
    return -1;
  }
  for (Py_ssize_t i = 0; i < len; i++) {
    long long v = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(f, i));
    if (v == -1 && PyErr_Occurred()) {
      Py_DECREF(f);
      return -1;
    }
    buf[i] = (int64_t)v;
  }
  *n = (int)len;
  Py_DECREF(f);
  return 0;
}

static PyObject* reduce(TensorObject* self, PyObject* axes, int op) {
  if (!has_handle(self)) return NULL;
  int64_t a[16];
  int n = 0;
  if (int64s(axes, a, &n)) return NULL;
  fg_tensor* out = NULL;
  if (fg_tensor_reduce(self->h, op, a, n, &out)) return raise_last();
  return wrap(Py_TYPE(self), out);
}

static PyObject* movement(TensorObject* self, PyObject* arg, int op) {
  if (!has_handle(self)) return NULL;
  int64_t a[16];
  int n = 0;
  if (int64s(arg, a, &n)) return NULL;
  fg_tensor* out = NULL;
  if (fg_tensor_movement(self->h, op, a, n, &out)) return raise_last();
  return wrap(Py_TYPE(self), out);
}

#define UNARY(name, op) \
  static PyObject* t_##name(TensorObject* self, PyObject* unused) { (void)unused; return unary(self, op); }
UNARY(neg, FG_UNARY_NEG)
UNARY(reciprocal, FG_UNARY_RECIPROCAL)
UNARY(exp2, FG_UNARY_EXP2)
UNARY(log2, FG_UNARY_LOG2)
UNARY(sqrt, FG_UNARY_SQRT)
UNARY(relu, FG_UNARY_RELU)
UNARY(exp, FG_UNARY_EXP)
UNARY(log, FG_UNARY_LOG)
UNARY(contiguous, FG_UNARY_CONTIGUOUS)
UNARY(detach, FG_UNARY_DETACH)
UNARY(alias, FG_UNARY_ALIAS)

#define BINARY(name, op) \
  static PyObject* t_##name(TensorObject* self, PyObject* other) { return binary(self, other, op); }
BINARY(add, FG_BINARY_ADD)
BINARY(mul, FG_BINARY_MUL)
BINARY(sub, FG_BINARY_SUB)
BINARY(matmul, FG_BINARY_MATMUL)
BINARY(cross_entropy, FG_BINARY_CROSS_ENTROPY)

static PyObject* t_sum(TensorObject* self, PyObject* axes) { return reduce(self, axes, FG_REDUCE_SUM); }
static PyObject* t_max(TensorObject* self, PyObject* axes) { return reduce(self, axes, FG_REDUCE_MAX); }
static PyObject* t_reshape(TensorObject* self, PyObject* s) { return movement(self, s, FG_MOVE_RESHAPE); }
static PyObject* t_permute(TensorObject* self, PyObject* s) { return movement(self, s, FG_MOVE_PERMUTE); }
static PyObject* t_expand(TensorObject* self, PyObject* s) { return movement(self, s, FG_MOVE_EXPAND); }

static PyObject* t_u(TensorObject* self, PyObject* op) {
  long v = PyLong_AsLong(op);
  if (v == -1 && PyErr_Occurred()) return NULL;
  return unary(self, (int)v);
}

static PyObject* t_b(TensorObject* self, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "_b(other, op)");
    return NULL;
  }
  long v = PyLong_AsLong(args[1]);
  if (v == -1 && PyErr_Occurred()) return NULL;
  return binary(self, args[0], (int)v);
}

static PyObject* t_narrow(TensorObject* self, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 3) {
    PyErr_SetString(PyExc_TypeError, "narrow(dim, start, length)");
    return NULL;
  }
  if (!has_handle(self)) return NULL;
  long long v[3];
  for (int i = 0; i < 3; i++) {
    v[i] = PyLong_AsLongLong(args[i]);
    if (v[i] == -1 && PyErr_Occurred()) return NULL;
  }
  fg_tensor* out = NULL;
  if (fg_tensor_narrow(self->h, v[0], v[1], v[2], &out)) return raise_last();
  return wrap(Py_TYPE(self), out);
}

static PyObject* t_log_softmax(TensorObject* self, PyObject* axis) {
  if (!has_handle(self)) return NULL;
  long long a = PyLong_AsLongLong(axis);
  if (a == -1 && PyErr_Occurred()) return NULL;
  fg_tensor* out = NULL;
  if (fg_tensor_log_softmax(self->h, a, &out)) return raise_last();
  return wrap(Py_TYPE(self), out);
}

PyDoc_STRVAR(attention_doc,
"attention(k, v, heads, kv_heads=None, batch=1, causal=False, lengths=None, scale=None)\n--\n\n"
"softmax(scale q k^T) v per head, with this tensor as q. Matrices have one row\n"
"per token, as Linear takes and gives them: q [batch * sq, heads * dim], k and v\n"
"[batch * sk, kv_heads * dim] (f32, dim at most 128); kv_heads defaults to heads,\n"
"scale to dim ** -0.5. Query i of a sequence sees the keys j < lengths[b] (an\n"
"int32 tensor [batch], clamped to [0, sk]; None: all of them) and, with causal,\n"
"j <= i + sk - sq; one that sees none gives 0 and gradients of 0. What keys and\n"
"values past a length hold never matters; everything else must be finite.");

static PyObject* t_attention(TensorObject* self, PyObject* args, PyObject* kw) {
  static char* names[] = {"k", "v", "heads", "kv_heads", "batch", "causal", "lengths", "scale", NULL};
  PyObject *kv_heads = Py_None, *lengths = Py_None, *scale = Py_None;
  TensorObject *k, *v, *l = NULL;
  PyObject *ko, *vo;
  long long heads, kvh, batch = 1;
  int causal = 0;
  if (!PyArg_ParseTupleAndKeywords(args, kw, "OOL|OLpOO:attention", names, &ko, &vo, &heads, &kv_heads, &batch, &causal,
                                   &lengths, &scale))
    return NULL;
  if (check_tensor(ko, &k) || check_tensor(vo, &v) || (lengths != Py_None && check_tensor(lengths, &l))) return NULL;
  if (!has_handle(self) || !has_handle(k) || !has_handle(v) || (l && !has_handle(l))) return NULL;
  kvh = heads;
  if (kv_heads != Py_None) {
    kvh = PyLong_AsLongLong(kv_heads);
    if (kvh == -1 && PyErr_Occurred()) return NULL;
  }
  double s = 1.0;
  if (scale != Py_None) {
    s = PyFloat_AsDouble(scale);
    if (s == -1.0 && PyErr_Occurred()) return NULL;
  } else {
    int64_t shape[16];
    int n = 16;
    if (fg_tensor_shape(self->h, shape, &n)) return raise_last();
    /* A shape that does not split is refused below. */
    if (n == 2 && heads > 0 && shape[1] >= heads) s = 1.0 / sqrt((double)(shape[1] / heads));
  }
  fg_tensor* out = NULL;
  if (fg_tensor_attention(self->h, k->h, v->h, l ? l->h : NULL, batch, heads, kvh, causal, s, &out)) return raise_last();
  return wrap(Py_TYPE(self), out);
}

PyDoc_STRVAR(norm_rotate_doc,
"norm_rotate(weight, positions, heads, eps=1e-6, base=10000.0)\n--\n\n"
"RMS norm of each head and the rotation of its position in one pass, for queries\n"
"and keys [tokens, heads * dim] (f32, dim even and at most 512): z = x *\n"
"(mean(x**2) + eps) ** -0.5 * weight (f32 [dim]), then the pair (z_i,\n"
"z_{i + dim/2}) turned by positions[token] * base**(-2i/dim) (positions int32\n"
"[tokens]).");

static PyObject* t_norm_rotate(TensorObject* self, PyObject* args, PyObject* kw) {
  static char* names[] = {"weight", "positions", "heads", "eps", "base", NULL};
  PyObject *wo, *po;
  TensorObject *w, *p;
  long long heads;
  double eps = 1e-6, base = 10000.0;
  if (!PyArg_ParseTupleAndKeywords(args, kw, "OOL|dd:norm_rotate", names, &wo, &po, &heads, &eps, &base)) return NULL;
  if (check_tensor(wo, &w) || check_tensor(po, &p) || !has_handle(self) || !has_handle(w) || !has_handle(p)) return NULL;
  fg_tensor* out = NULL;
  if (fg_tensor_norm_rotate(self->h, w->h, p->h, heads, eps, base, &out)) return raise_last();
  return wrap(Py_TYPE(self), out);
}

PyDoc_STRVAR(dropout_doc,
"dropout(p, seed, offset=0)\n--\n\n"
"x / (1 - p) where the element's random word is at least floor(p * 2**32), else\n"
"0 (an f32 tensor of any shape; 0 <= p < 1). Element e's word is word e % 4 of\n"
"Philox4x32-10 of the counter (e // 4, offset) under the key `seed`: 64 bits\n"
"each, so the same seed and offset drop the same elements, and the gradient draws\n"
"the mask again. Use a new offset for every call that should draw anew (Dropout\n"
"does).");

/* An int of [0, 2^64). */
static int u64_arg(PyObject* o, const char* name, uint64_t* out) {
  PyObject* i = PyNumber_Index(o);
  if (!i) return -1;
  *out = PyLong_AsUnsignedLongLong(i);
  if (*out == (uint64_t)-1 && PyErr_Occurred()) {
    PyErr_Clear();
    PyErr_Format(g_error_class ? g_error_class : PyExc_RuntimeError, "%s must be in [0, 2**64), got %S", name, i);
    Py_DECREF(i);
    return -1;
  }
  Py_DECREF(i);
  return 0;
}

static PyObject* t_dropout(TensorObject* self, PyObject* args, PyObject* kw) {
  static char* names[] = {"p", "seed", "offset", NULL};
  PyObject *so, *oo = NULL;
  double p;
  uint64_t seed, offset = 0;
  if (!PyArg_ParseTupleAndKeywords(args, kw, "dO|O:dropout", names, &p, &so, &oo)) return NULL;
  if (u64_arg(so, "seed", &seed) || (oo && u64_arg(oo, "offset", &offset)) || !has_handle(self)) return NULL;
  fg_tensor* out = NULL;
  if (fg_tensor_dropout(self->h, p, seed, offset, &out)) return raise_last();
  return wrap(Py_TYPE(self), out);
}

PyDoc_STRVAR(embedding_doc,
"embedding(ids, scale=1.0)\n--\n\n"
"Rows of this weight [vocab, dim] (f32) by id, times scale: [tokens, dim] of ids\n"
"(an int32 tensor [tokens]). An id outside of [0, vocab) is no token: a row of\n"
"zeros, and no gradient. The weight's gradient sums its tokens' rows in an order\n"
"fixed by the ids and the sizes: the same in every run.");

static PyObject* t_embedding(TensorObject* self, PyObject* args, PyObject* kw) {
  static char* names[] = {"ids", "scale", NULL};
  PyObject* io;
  TensorObject* ids;
  double scale = 1.0;
  if (!PyArg_ParseTupleAndKeywords(args, kw, "O|d:embedding", names, &io, &scale)) return NULL;
  if (check_tensor(io, &ids) || !has_handle(self) || !has_handle(ids)) return NULL;
  fg_tensor* out = NULL;
  if (fg_tensor_embedding(self->h, ids->h, scale, &out)) return raise_last();
  return wrap(Py_TYPE(self), out);
}

PyDoc_STRVAR(layer_norm_doc,
"layer_norm(weight, bias=None, eps=1e-5)\n--\n\n"
"Layer norm of each row [rows, dim] (f32): (x - mean) / sqrt(variance + eps) *\n"
"weight + bias, with weight and bias f32 [dim] (bias None: none).");

static PyObject* t_layer_norm(TensorObject* self, PyObject* args, PyObject* kw) {
  static char* names[] = {"weight", "bias", "eps", NULL};
  PyObject *wo, *bo = Py_None;
  TensorObject *w, *b = NULL;
  double eps = 1e-5;
  if (!PyArg_ParseTupleAndKeywords(args, kw, "O|Od:layer_norm", names, &wo, &bo, &eps)) return NULL;
  if (check_tensor(wo, &w) || (bo != Py_None && check_tensor(bo, &b))) return NULL;
  if (!has_handle(self) || !has_handle(w) || (b && !has_handle(b))) return NULL;
  fg_tensor* out = NULL;
  if (fg_tensor_layer_norm(self->h, w->h, b ? b->h : NULL, eps, &out)) return raise_last();
  return wrap(Py_TYPE(self), out);
}

PyDoc_STRVAR(token_cross_entropy_doc,
"token_cross_entropy(labels)\n--\n\n"
"The mean of logsumexp(row) - row[label] over the rows of these logits [rows,\n"
"classes] (f32) whose label (an int32 tensor [rows]) is in [0, classes), as a\n"
"tensor [1]. Rows of other labels are ignored and get gradients of 0; a loss of 0\n"
"where all are. With every label valid it is cross_entropy of one-hot rows, which\n"
"need not be made. Logits of -inf are classes that a row cannot take; a row of\n"
"nothing else, or with a NaN or +inf, makes the loss and its own gradients NaN.");

static PyObject* t_token_cross_entropy(TensorObject* self, PyObject* args, PyObject* kw) {
  static char* names[] = {"labels", NULL};
  PyObject* lo;
  TensorObject* labels;
  if (!PyArg_ParseTupleAndKeywords(args, kw, "O:token_cross_entropy", names, &lo)) return NULL;
  if (check_tensor(lo, &labels) || !has_handle(self) || !has_handle(labels)) return NULL;
  fg_tensor* out = NULL;
  if (fg_tensor_token_cross_entropy(self->h, labels->h, &out)) return raise_last();
  return wrap(Py_TYPE(self), out);
}

static PyObject* t_realize(TensorObject* self, PyObject* unused) {
  (void)unused;
  if (!has_handle(self)) return NULL;
  if (fg_tensor_realize_many(&self->h, 1)) return raise_last();
  Py_INCREF(self);
  return (PyObject*)self;
}

static PyObject* t_assign(TensorObject* self, PyObject* other) {
  TensorObject* o;
  if (check_tensor(other, &o) || !has_handle(self) || !has_handle(o)) return NULL;
  if (fg_tensor_assign(self->h, o->h)) return raise_last();
  Py_INCREF(self);
  return (PyObject*)self;
}

/* The handles of a sequence of Tensors (and room for as many more behind them),
 * with a tuple that keeps the tensors, whatever another thread does to a list of
 * them: free_handles returns both. */
static fg_tensor** handles_of(PyObject* tensors, PyObject** seq, int* n) {
  *seq = PySequence_Tuple(tensors);
  if (!*seq) return NULL;
  const Py_ssize_t count = PyTuple_GET_SIZE(*seq);
  fg_tensor** hs = count <= INT_MAX ? PyMem_New(fg_tensor*, 2 * (size_t)count + 1) : NULL;
  if (!hs) {
    Py_DECREF(*seq);
    return (fg_tensor**)PyErr_NoMemory();
  }
  for (Py_ssize_t i = 0; i < count; i++) {
    TensorObject* t;
    if (check_tensor(PyTuple_GET_ITEM(*seq, i), &t) || !has_handle(t)) {
      PyMem_Free(hs);
      Py_DECREF(*seq);
      return NULL;
    }
    hs[i] = t->h;
  }
  *n = (int)count;
  return hs;
}

static void free_handles(fg_tensor** hs, PyObject* seq) {
  PyMem_Free(hs);
  Py_DECREF(seq);
}

/* A list of objects of `tp` owning the handles; what is not wrapped is freed. */
static PyObject* wrap_list(PyTypeObject* tp, fg_tensor** hs, int n) {
  PyObject* list = PyList_New(n);
  for (int i = 0; i < n; i++) {
    PyObject* t = list ? wrap(tp, hs[i]) : NULL;
    if (!list) fg_tensor_free(hs[i]);
    else if (!t) Py_CLEAR(list); /* wrap freed this one */
    else PyList_SET_ITEM(list, i, t);
  }
  return list;
}

/* The one argument of `func`, by position or as `name`. */
static PyObject* one_argument(const char* func, const char* name, PyObject* const* args, Py_ssize_t n, PyObject* kwnames) {
  const Py_ssize_t named = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
  if (n + named != 1) {
    PyErr_Format(PyExc_TypeError, "%s() takes exactly one argument (%zd given)", func, n + named);
  } else if (named && PyUnicode_CompareWithASCIIString(PyTuple_GET_ITEM(kwnames, 0), name) != 0) {
    PyErr_Format(PyExc_TypeError, "%s() got an unexpected keyword argument '%U'", func, PyTuple_GET_ITEM(kwnames, 0));
  } else {
    return args[0];
  }
  return NULL;
}

PyDoc_STRVAR(realize_many_doc, "realize_many(tensors)\n--\n\nTensor::realize_many (tensor.rs:781-830).");

static PyObject* t_realize_many(PyObject* unused, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  (void)unused;
  PyObject* seq;
  int n;
  PyObject* tensors = one_argument("realize_many", "tensors", args, nargs, kwnames);
  fg_tensor** hs = tensors ? handles_of(tensors, &seq, &n) : NULL;
  if (!hs) return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fg_tensor_realize_many(hs, n);
  Py_END_ALLOW_THREADS
  free_handles(hs, seq);
  if (rc) return raise_last();
  Py_RETURN_NONE;
}

PyDoc_STRVAR(gradient_doc, "gradient($self, targets)\n--\n\nTensor::gradient (tensor.rs:938-964): the list of d self / d target.");

static PyObject* t_gradient(TensorObject* self, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  PyObject* seq;
  int n;
  PyObject* targets = one_argument("gradient", "targets", args, nargs, kwnames);
  if (!targets || !has_handle(self)) return NULL;
  fg_tensor** hs = handles_of(targets, &seq, &n);
  if (!hs) return NULL;
  PyObject* list = NULL;
  fg_tensor* const h = self->h;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fg_tensor_gradient(h, hs, n, hs + n);
  Py_END_ALLOW_THREADS
  if (rc) raise_last();
  else list = wrap_list(Py_TYPE(self), hs + n, n);
  free_handles(hs, seq);
  return list;
}

PyDoc_STRVAR(data_ptr_doc, "data_ptr()\n--\n\n(device pointer, byte size) of a realised tensor's storage.");

static PyObject* t_data_ptr(TensorObject* self, PyObject* unused) {
  (void)unused;
  void* p = NULL;
  size_t nbytes = 0;
  if (!has_handle(self)) return NULL;
  if (fg_tensor_data_ptr(self->h, &p, &nbytes)) return raise_last();
  return Py_BuildValue("(NN)", p ? PyLong_FromVoidPtr(p) : Py_NewRef(Py_None), PyLong_FromSize_t(nbytes));
}

static PyObject* t_get_shape(TensorObject* self, void* closure) {
  (void)closure;
  int64_t shape[16];
  int n = 16;
  if (!has_handle(self)) return NULL;
  if (fg_tensor_shape(self->h, shape, &n)) return raise_last();
  PyObject* t = PyTuple_New(n);
  for (int i = 0; t && i < n; i++) {
    PyObject* d = PyLong_FromLongLong(shape[i]);
    if (!d) Py_CLEAR(t);
    else PyTuple_SET_ITEM(t, i, d);
  }
  return t;
}

static PyMethodDef t_methods[] = {
    {"neg", (PyCFunction)t_neg, METH_NOARGS, NULL},
    {"reciprocal", (PyCFunction)t_reciprocal, METH_NOARGS, NULL},
    {"exp2", (PyCFunction)t_exp2, METH_NOARGS, NULL},
    {"log2", (PyCFunction)t_log2, METH_NOARGS, NULL},
    {"sqrt", (PyCFunction)t_sqrt, METH_NOARGS, NULL},
    {"relu", (PyCFunction)t_relu, METH_NOARGS, NULL},
    {"exp", (PyCFunction)t_exp, METH_NOARGS, NULL},
    {"log", (PyCFunction)t_log, METH_NOARGS, NULL},
    {"contiguous", (PyCFunction)t_contiguous, METH_NOARGS, NULL},
    {"detach", (PyCFunction)t_detach, METH_NOARGS, NULL},
    {"alias", (PyCFunction)t_alias, METH_NOARGS, "A second handle to the same tensor identity (a Rust `clone`)."},
    {"add", (PyCFunction)t_add, METH_O, NULL},
    {"mul", (PyCFunction)t_mul, METH_O, NULL},
    {"sub", (PyCFunction)t_sub, METH_O, NULL},
    {"matmul", (PyCFunction)t_matmul, METH_O, NULL},
    {"cross_entropy", (PyCFunction)t_cross_entropy, METH_O, NULL},
    {"sum", (PyCFunction)t_sum, METH_O, NULL},
    {"max", (PyCFunction)t_max, METH_O, NULL},
    {"reshape", (PyCFunction)t_reshape, METH_O, NULL},
    {"permute", (PyCFunction)t_permute, METH_O, NULL},
    {"expand", (PyCFunction)t_expand, METH_O, NULL},
    {"narrow", (PyCFunction)(void (*)(void))t_narrow, METH_FASTCALL, NULL},
    {"log_softmax", (PyCFunction)t_log_softmax, METH_O, NULL},
    {"attention", (PyCFunction)(void (*)(void))t_attention, METH_VARARGS | METH_KEYWORDS, attention_doc},
    {"norm_rotate", (PyCFunction)(void (*)(void))t_norm_rotate, METH_VARARGS | METH_KEYWORDS, norm_rotate_doc},
    {"dropout", (PyCFunction)(void (*)(void))t_dropout, METH_VARARGS | METH_KEYWORDS, dropout_doc},
    {"embedding", (PyCFunction)(void (*)(void))t_embedding, METH_VARARGS | METH_KEYWORDS, embedding_doc},
    {"layer_norm", (PyCFunction)(void (*)(void))t_layer_norm, METH_VARARGS | METH_KEYWORDS, layer_norm_doc},
    {"token_cross_entropy", (PyCFunction)(void (*)(void))t_token_cross_entropy, METH_VARARGS | METH_KEYWORDS,
     token_cross_entropy_doc},
    {"_u", (PyCFunction)t_u, METH_O, NULL},
    {"_b", (PyCFunction)(void (*)(void))t_b, METH_FASTCALL, NULL},
    {"realize", (PyCFunction)t_realize, METH_NOARGS, "Tensor::realize (tensor.rs:781-830)."},
    {"assign", (PyCFunction)t_assign, METH_O, "Tensor::assign (tensor.rs:421-440)."},
    {"realize_many", (PyCFunction)(void (*)(void))t_realize_many, METH_FASTCALL | METH_KEYWORDS | METH_STATIC, realize_many_doc},
    {"gradient", (PyCFunction)(void (*)(void))t_gradient, METH_FASTCALL | METH_KEYWORDS, gradient_doc},
    {"data_ptr", (PyCFunction)t_data_ptr, METH_NOARGS, data_ptr_doc},
    {NULL, NULL, 0, NULL},
};

static PyGetSetDef t_getset[] = {
    {"_h", (getter)t_get_h, NULL, "the fg_tensor handle, as an int (None when empty)", NULL},
    {"shape", (getter)t_get_shape, NULL, "the shape, as a tuple", NULL},
    {NULL, NULL, NULL, NULL, NULL},
};

static PyTypeObject TensorBaseType = {
    PyVarObject_HEAD_INIT(NULL, 0).tp_name = "ferrograd_amd._fgc.TensorBase",
    .tp_basicsize = sizeof(TensorObject),
    .tp_dealloc = (destructor)t_dealloc,
    .tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_BASETYPE,
    .tp_doc = "A lazily evaluated tensor handle (tensor.rs:95-97); the hot ops in C.",
    .tp_weaklistoffset = offsetof(TensorObject, weakrefs),
    .tp_methods = t_methods,
    .tp_getset = t_getset,
    .tp_init = (initproc)t_init,
    .tp_new = PyType_GenericNew,
};

static int check_tensor(PyObject* o, TensorObject** out) {
  if (!PyObject_TypeCheck(o, &TensorBaseType)) {
    PyErr_SetString(PyExc_TypeError, "expected a Tensor");
    return -1;
  }
  *out = (TensorObject*)o;
  return 0;
}

/* from_handle(cls, h): a `cls` owning handle h (an int). */
static PyObject* m_from_handle(PyObject* mod, PyObject* const* args, Py_ssize_t nargs) {
  (void)mod;
  if (nargs != 2 || !PyType_Check(args[0]) || !PyType_IsSubtype((PyTypeObject*)args[0], &TensorBaseType)) {
    PyErr_SetString(PyExc_TypeError, "from_handle(Tensor subclass, handle)");
    return NULL;
  }
  void* p = PyLong_AsVoidPtr(args[1]);
  if (!p) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null tensor handle");
    return NULL;
  }
  return wrap((PyTypeObject*)args[0], (fg_tensor*)p);
}

static PyObject* m_set_error_class(PyObject* mod, PyObject* cls) {
  (void)mod;
  Py_XINCREF(cls);
  Py_XSETREF(g_error_class, cls);
  Py_RETURN_NONE;
}

/* global_norm(cls, tensors): a `cls`. */
static PyObject* m_global_norm(PyObject* mod, PyObject* args) {
  (void)mod;
  PyTypeObject* cls;
  PyObject *tensors, *seq;
  int n;
  if (!PyArg_ParseTuple(args, "O!O:global_norm", &PyType_Type, &cls, &tensors)) return NULL;
  fg_tensor** hs = handles_of(tensors, &seq, &n);
  if (!hs) return NULL;
  fg_tensor* norm = NULL;
  const int rc = fg_global_norm(hs, n, &norm);
  free_handles(hs, seq);
  return rc ? raise_last() : wrap(cls, norm);
}

/* clip_norm(cls, tensors, max_norm): (a `cls`, a list of them). */
static PyObject* m_clip_norm(PyObject* mod, PyObject* args) {
  (void)mod;
  PyTypeObject* cls;
  PyObject *tensors, *seq;
  double max_norm;
  int n;
  if (!PyArg_ParseTuple(args, "O!Od:clip_norm", &PyType_Type, &cls, &tensors, &max_norm)) return NULL;
  fg_tensor** hs = handles_of(tensors, &seq, &n);
  if (!hs) return NULL;
  fg_tensor* norm = NULL;
  PyObject* out = NULL;
  if (fg_clip_norm(hs, n, max_norm, &norm, hs + n)) {
    raise_last();
  } else {
    PyObject* list = wrap_list(cls, hs + n, n);
    PyObject* t = wrap(cls, norm);
    if (list && t) out = PyTuple_Pack(2, t, list);
    Py_XDECREF(t);
    Py_XDECREF(list);
  }
  free_handles(hs, seq);
  return out;
}

static PyMethodDef m_methods[] = {
    {"global_norm", m_global_norm, METH_VARARGS, NULL},
    {"clip_norm", m_clip_norm, METH_VARARGS, NULL},
    {"from_handle", (PyCFunction)(void (*)(void))m_from_handle, METH_FASTCALL, NULL},
    {"set_error_class", (PyCFunction)m_set_error_class, METH_O, NULL},
    {NULL, NULL, 0, NULL},
};

static struct PyModuleDef fgc_module = {PyModuleDef_HEAD_INIT, "_fgc", NULL, -1, m_methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__fgc(void) {
  if (PyType_Ready(&TensorBaseType) < 0) return NULL;
  PyObject* m = PyModule_Create(&fgc_module);
  if (!m) return NULL;
  Py_INCREF(&TensorBaseType);
  if (PyModule_AddObject(m, "TensorBase", (PyObject*)&TensorBaseType) < 0) {
    Py_DECREF(&TensorBaseType);
    Py_DECREF(m);
    return NULL;
  }
  return m;
}
