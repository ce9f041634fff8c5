/*
 * Plain group calls from Python: checks the tensors of a call against the
 * group's manifest and launches, in one C function.
 *
 * A kernel of a few microseconds waits for its call: looked up and packed in
 * Python, six tensors and the launch took 6.8 us of host time, of which 2.7
 * were the checks and the packing and about 0.7 the foreign call.  The checks
 * are the ones the Python path makes (a torch.Tensor on the GPU, the group's
 * element type and shape, contiguous); a call that does not pass them returns
 * None and the Python path says why.  Tensors are read through their public
 * Python attributes, so this file needs nothing of torch to build.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>
#include <structmember.h>

typedef int (*launch_fn)(void *, const uint64_t *, size_t, void *const *, size_t, void *, void *);
typedef int (*launch_rows_fn)(void *, const uint64_t *, size_t, void *const *, size_t, int64_t, void *, void *);

#define MAX_ARGS 24
#define MAX_RANK 8

static PyObject *s_dtype, *s_is_cuda, *s_shape, *s_is_contiguous, *s_data_ptr, *s_get_device;

typedef struct {
  PyObject *dtype;
  int rank;
  int64_t shape[MAX_RANK]; /* -1: the launch-time row count */
} Spec;

typedef struct {
  PyObject_HEAD
  vectorcallfunc call;
  PyObject *tensor_type, *raw_stream, *capturing; /* capturing: None, or asked before a call that takes the group's workspace */
  void *fn, *handle;
  int n, nres, dyn;
  Spec spec[MAX_ARGS];
  int tied[MAX_ARGS];
} Call;

/* 1: the argument passes and *ptr is set; 0: it does not; -1: a Python error */
static int take(const Spec *sp, PyObject *a, int64_t *rows, uint64_t *ptr) {
  PyObject *v = PyObject_GetAttr(a, s_dtype);
  if (!v) return -1;
  const int same = v == sp->dtype;
  Py_DECREF(v);
  if (!same) return 0;
  if (!(v = PyObject_GetAttr(a, s_is_cuda))) return -1;
  const int cuda = v == Py_True;
  Py_DECREF(v);
  if (!cuda) return 0;
  if (!(v = PyObject_GetAttr(a, s_shape))) return -1;
  int ok = PyTuple_Check(v) && PyTuple_GET_SIZE(v) == sp->rank;
  for (int d = 0; ok && d < sp->rank; ++d) {
    const long long x = PyLong_AsLongLong(PyTuple_GET_ITEM(v, d));
    if (x < 0) ok = 0;
    else if (sp->shape[d] >= 0) ok = x == sp->shape[d];
    else if (*rows < 0) *rows = x;
    else ok = x == *rows;
  }
  Py_DECREF(v);
  if (PyErr_Occurred()) return -1;
  if (!ok) return 0;
  if (!(v = PyObject_CallMethodNoArgs(a, s_is_contiguous))) return -1;
  const int dense = v == Py_True;
  Py_DECREF(v);
  if (!dense) return 0;
  if (!(v = PyObject_CallMethodNoArgs(a, s_data_ptr))) return -1;
  *ptr = PyLong_AsUnsignedLongLong(v);
  Py_DECREF(v);
  return PyErr_Occurred() ? -1 : 1;
}

static PyObject *call_call(PyObject *self, PyObject *const *args, size_t nargsf, PyObject *kwnames) {
  Call *c = (Call *)self;
  if (PyVectorcall_NARGS(nargsf) != c->n || (kwnames && PyTuple_GET_SIZE(kwnames))) Py_RETURN_NONE;
  if (c->capturing != Py_None) {
    PyObject *v = PyObject_CallNoArgs(c->capturing);
    if (!v) return NULL;
    const int yes = v == Py_True;
    Py_DECREF(v);
    if (yes) Py_RETURN_NONE; /* (the graph's own workspace: the Python path's work) */
  }
  uint64_t slots[MAX_ARGS];
  void *results[MAX_ARGS] = {0}; /* every result is written into an argument */
  int64_t rows = -1;
  for (int i = 0; i < c->n; ++i) {
    if ((PyObject *)Py_TYPE(args[i]) != c->tensor_type) Py_RETURN_NONE;
    const int r = take(&c->spec[i], args[i], &rows, &slots[i]);
    if (r < 0) return NULL;
    if (r == 0) Py_RETURN_NONE;
  }
  PyObject *dev = PyObject_CallMethodNoArgs(args[0], s_get_device);
  if (!dev) return NULL;
  PyObject *st = PyObject_CallOneArg(c->raw_stream, dev);
  Py_DECREF(dev);
  if (!st) return NULL;
  void *stream = PyLong_AsVoidPtr(st);
  Py_DECREF(st);
  if (PyErr_Occurred()) return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (c->dyn) rc = ((launch_rows_fn)c->fn)(c->handle, slots, (size_t)c->n, results, (size_t)c->nres, rows, NULL, stream);
  else rc = ((launch_fn)c->fn)(c->handle, slots, (size_t)c->n, results, (size_t)c->nres, NULL, stream);
  Py_END_ALLOW_THREADS
  if (rc) return PyLong_FromLong(rc);
  if (c->nres == 1) {
    Py_INCREF(args[c->tied[0]]);
    return args[c->tied[0]];
  }
  PyObject *out = PyTuple_New(c->nres);
  if (!out) return NULL;
  for (int i = 0; i < c->nres; ++i) {
    Py_INCREF(args[c->tied[i]]);
    PyTuple_SET_ITEM(out, i, args[c->tied[i]]);
  }
  return out;
}

static void call_dealloc(PyObject *self) {
  Call *c = (Call *)self;
  for (int i = 0; i < c->n; ++i) Py_XDECREF(c->spec[i].dtype);
  Py_XDECREF(c->tensor_type);
  Py_XDECREF(c->raw_stream);
  Py_XDECREF(c->capturing);
  Py_TYPE(self)->tp_free(self);
}

static PyTypeObject CallType = {
    PyVarObject_HEAD_INIT(NULL, 0).tp_name = "_hfcall.Call",
    .tp_basicsize = sizeof(Call),
    .tp_dealloc = call_dealloc,
    .tp_vectorcall_offset = offsetof(Call, call),
    .tp_call = PyVectorcall_Call,
    .tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL,
    .tp_doc = "The plain call of one group: call(*tensors) launches and returns the result (or results), "
              "None where the arguments are not what the group takes, or the launch's error code.",
};

/* plan(launch address, handle, launch takes rows, torch.Tensor, stream getter,
 *      ((dtype, shape), ...) per argument, tied argument per result, capture query) */
static PyObject *plan(PyObject *self, PyObject *args) {
  (void)self;
  unsigned long long fn, handle;
  int dyn;
  PyObject *tensor_type, *raw_stream, *specs, *tied, *capturing = Py_None;
  if (!PyArg_ParseTuple(args, "KKpOOO!O!|O", &fn, &handle, &dyn, &tensor_type, &raw_stream, &PyTuple_Type, &specs, &PyTuple_Type, &tied,
                        &capturing))
    return NULL;
  const Py_ssize_t n = PyTuple_GET_SIZE(specs), nres = PyTuple_GET_SIZE(tied);
  if (n < 1 || n > MAX_ARGS || nres < 1 || nres > MAX_ARGS || !fn || !handle) {
    PyErr_SetString(PyExc_ValueError, "arguments or results out of range");
    return NULL;
  }
  Call *c = PyObject_New(Call, &CallType);
  if (!c) return NULL;
  c->call = call_call;
  c->n = 0;
  c->tensor_type = c->raw_stream = c->capturing = NULL;
  c->fn = (void *)(uintptr_t)fn;
  c->handle = (void *)(uintptr_t)handle;
  c->dyn = dyn;
  c->nres = (int)nres;
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject *dtype, *shape;
    Spec *sp = &c->spec[i];
    if (!PyArg_ParseTuple(PyTuple_GET_ITEM(specs, i), "OO!", &dtype, &PyTuple_Type, &shape)) goto fail;
    if (PyTuple_GET_SIZE(shape) > MAX_RANK) {
      PyErr_SetString(PyExc_ValueError, "rank out of range");
      goto fail;
    }
    sp->rank = (int)PyTuple_GET_SIZE(shape);
    for (int d = 0; d < sp->rank; ++d) sp->shape[d] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, d));
    if (PyErr_Occurred()) goto fail;
    Py_INCREF(dtype);
    sp->dtype = dtype;
    c->n = (int)i + 1;
  }
  for (Py_ssize_t i = 0; i < nres; ++i) {
    const long t = PyLong_AsLong(PyTuple_GET_ITEM(tied, i));
    if (PyErr_Occurred()) goto fail;
    if (t < 0 || t >= n) {
      PyErr_SetString(PyExc_ValueError, "a result that is not written into an argument");
      goto fail;
    }
    c->tied[i] = (int)t;
  }
  Py_INCREF(tensor_type);
  Py_INCREF(raw_stream);
  Py_INCREF(capturing);
  c->tensor_type = tensor_type;
  c->raw_stream = raw_stream;
  c->capturing = capturing;
  return (PyObject *)c;
fail:
  Py_DECREF(c);
  return NULL;
}

static PyMethodDef methods[] = {{"plan", plan, METH_VARARGS, "The plain call of a group (see _hfcall.Call)."}, {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hfcall", "Plain group calls.", -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__hfcall(void) {
  if (PyType_Ready(&CallType) < 0) return NULL;
  const char *names[] = {"dtype", "is_cuda", "shape", "is_contiguous", "data_ptr", "get_device"};
  PyObject **slots[] = {&s_dtype, &s_is_cuda, &s_shape, &s_is_contiguous, &s_data_ptr, &s_get_device};
  for (int i = 0; i < 6; ++i)
    if (!(*slots[i] = PyUnicode_InternFromString(names[i]))) return NULL;
  return PyModule_Create(&module);
}
