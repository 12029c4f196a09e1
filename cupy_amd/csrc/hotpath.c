/* CPython extension for the calls the host makes per kernel launch:
 * the signature of its arguments (the key a recorded call is found by), the
 * launch itself, the replay of a recorded call, and the memory pool's
 * malloc/free.  Each is a thin caller of the C-ABI in include/mi355rt.h
 * (rt_launch_packed, rt_pool_malloc, rt_pool_free); what it removes is the
 * per-argument conversion cost of a ctypes call (about 1 us for the eleven
 * arguments of a launch) and the interpreter loop that splices pointers into a
 * recorded argument block.  The reference does this part of the path in
 * compiled Cython (cupy/_core/_kernel.pyx:166-247 argument packing,
 * cupy/cuda/function.pyx:191-236 launch, cupy/cuda/memory.pyx:1373-1441 pool).
 *
 * Nothing here touches the GPU on its own: every GPU effect goes through the
 * C-ABI, so the library and this module cannot disagree about it.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>

#include "mi355rt.h"

static PyObject* str_data;
static PyObject* str_ptr;
static PyObject* str_dtype;
static PyObject* str_shape;
static PyObject* str_strides;
static PyObject* str_device_id;
static PyObject* str_size;
static PyObject* str_itemsize;
static PyObject* str_c_contiguous;
static PyObject* str_f_contiguous;
static PyTypeObject* array_type;      /* the package's ndarray, set by setup() */
static PyTypeObject* generic_type;    /* numpy.generic */

static int as_u64(PyObject* o, uint64_t* out) {
  unsigned long long v = PyLong_AsUnsignedLongLong(o);
  if (v == (unsigned long long)-1 && PyErr_Occurred()) return -1;
  *out = (uint64_t)v;
  return 0;
}

static int as_u32(PyObject* o, unsigned* out) {
  unsigned long v = PyLong_AsUnsignedLong(o);
  if (v == (unsigned long)-1 && PyErr_Occurred()) return -1;
  if (v > 0xfffffffful) {
    PyErr_SetString(PyExc_OverflowError, "launch dimension does not fit 32 bits");
    return -1;
  }
  *out = (unsigned)v;
  return 0;
}

/* launch(function, gx, gy, gz, bx, by, bz, shared_mem, stream, arg_block) -> status */
static PyObject* hp_launch(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 10) {
    PyErr_SetString(PyExc_TypeError, "launch takes 10 arguments");
    return NULL;
  }
  uint64_t fn, stream;
  unsigned d[7];
  if (as_u64(args[0], &fn) < 0) return NULL;
  for (int i = 0; i < 7; ++i)
    if (as_u32(args[1 + i], &d[i]) < 0) return NULL;
  if (as_u64(args[8], &stream) < 0) return NULL;
  Py_buffer view;
  if (PyObject_GetBuffer(args[9], &view, PyBUF_SIMPLE) < 0) return NULL;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = rt_launch_packed((void*)(uintptr_t)fn, d[0], d[1], d[2], d[3], d[4], d[5], d[6],
                            (void*)(uintptr_t)stream, view.buf, (size_t)view.len);
  Py_END_ALLOW_THREADS
  PyBuffer_Release(&view);
  return PyLong_FromLong(status);
}

/* A recorded call, as one bytes object:
 *   u32 n_launches, u32 0
 *   per launch (8-byte aligned):
 *     u64 function, u32 grid[3], u32 block[3], u32 shared_mem, u32 n_slots,
 *     u64 block_size, then n_slots x (u32 byte offset, u32 ref), padded to 8,
 *     then the argument block, padded to 8.
 * A slot names the 8 bytes of the block that receive the device address of
 * refs[ref]: of its `.data.ptr` for ref < n_arrays (an array), of its `.ptr`
 * otherwise (a temporary's memory pointer). */
typedef struct {
  uint64_t function;
  uint32_t grid[3];
  uint32_t block[3];
  uint32_t shared_mem;
  uint32_t n_slots;
  uint64_t block_size;
} LaunchHeader;

#define HP_STACK_BLOCK 4096

static int address_of(PyObject* ref, int is_array, uint64_t* out) {
  PyObject* holder = ref;
  PyObject* data = NULL;
  if (is_array) {
    data = PyObject_GetAttr(ref, str_data);
    if (!data) return -1;
    holder = data;
  }
  PyObject* ptr = PyObject_GetAttr(holder, str_ptr);
  Py_XDECREF(data);
  if (!ptr) return -1;
  int rc = as_u64(ptr, out);
  Py_DECREF(ptr);
  return rc;
}

/* Walks a launch record: patches every argument block and either launches it
 * (`listing` NULL; returns the first non-zero status as an int object, else 0)
 * or appends (function, grid, block, shared_mem, patched block) to `listing`. */
static PyObject* walk_record(PyObject* record, PyObject* refs, long n_arrays, uint64_t stream,
                             PyObject* listing) {
  const unsigned char* rec = (const unsigned char*)PyBytes_AS_STRING(record);
  const size_t rec_size = (size_t)PyBytes_GET_SIZE(record);
  const Py_ssize_t n_refs = PyList_GET_SIZE(refs);
  unsigned char stack_block[HP_STACK_BLOCK] __attribute__((aligned(16)));
  uint32_t n_launches;
  size_t pos = 8;
  if (rec_size < 8) goto malformed;
  memcpy(&n_launches, rec, 4);
  for (uint32_t l = 0; l < n_launches; ++l) {
    LaunchHeader h;
    if (pos + sizeof(h) > rec_size) goto malformed;
    memcpy(&h, rec + pos, sizeof(h));
    pos += sizeof(h);
    const size_t slot_bytes = ((size_t)h.n_slots * 8 + 7) & ~(size_t)7;
    const size_t block_bytes = ((size_t)h.block_size + 7) & ~(size_t)7;
    if (slot_bytes > rec_size || block_bytes > rec_size ||
        pos + slot_bytes + block_bytes > rec_size)
      goto malformed;
    const unsigned char* slots = rec + pos;
    pos += slot_bytes;
    unsigned char* block = stack_block;
    if (h.block_size > HP_STACK_BLOCK) {
      block = (unsigned char*)PyMem_Malloc((size_t)h.block_size);
      if (!block) return PyErr_NoMemory();
    }
    memcpy(block, rec + pos, (size_t)h.block_size);
    pos += block_bytes;
    int bad = 0;
    for (uint32_t s = 0; s < h.n_slots; ++s) {
      uint32_t off, ref;
      memcpy(&off, slots + 8 * s, 4);
      memcpy(&ref, slots + 8 * s + 4, 4);
      if ((size_t)off + 8 > h.block_size || (Py_ssize_t)ref >= n_refs) {
        bad = 2;
        break;
      }
      uint64_t address;
      if (address_of(PyList_GET_ITEM(refs, ref), (long)ref < n_arrays, &address) < 0) {
        bad = 1;
        break;
      }
      memcpy(block + off, &address, 8);
    }
    int status = 0;
    if (!bad && listing) {
      PyObject* entry = Py_BuildValue(
          "K(III)(III)Iy#", (unsigned long long)h.function, h.grid[0], h.grid[1], h.grid[2],
          h.block[0], h.block[1], h.block[2], h.shared_mem, (const char*)block,
          (Py_ssize_t)h.block_size);
      if (!entry || PyList_Append(listing, entry) < 0) bad = 1;
      Py_XDECREF(entry);
    } else if (!bad) {
      Py_BEGIN_ALLOW_THREADS
      status = rt_launch_packed((void*)(uintptr_t)h.function, h.grid[0], h.grid[1], h.grid[2],
                                h.block[0], h.block[1], h.block[2], h.shared_mem,
                                (void*)(uintptr_t)stream, block, (size_t)h.block_size);
      Py_END_ALLOW_THREADS
    }
    if (block != stack_block) PyMem_Free(block);
    if (bad == 1) return NULL;
    if (bad == 2) goto malformed;
    if (status != 0) return PyLong_FromLong(status);
  }
  return PyLong_FromLong(0);
malformed:
  PyErr_SetString(PyExc_ValueError, "malformed launch record");
  return NULL;
}

/* replay(record, refs, n_arrays, stream) -> status of the first launch that failed, or 0 */
static PyObject* hp_replay(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 4 || !PyBytes_Check(args[0]) || !PyList_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "replay(record: bytes, refs: list, n_arrays, stream)");
    return NULL;
  }
  const long n_arrays = PyLong_AsLong(args[2]);
  if (n_arrays == -1 && PyErr_Occurred()) return NULL;
  uint64_t stream;
  if (as_u64(args[3], &stream) < 0) return NULL;
  return walk_record(args[0], args[1], n_arrays, stream, NULL);
}

/* splice(record, refs, n_arrays) -> [(function, grid, block, shared_mem, argument block)]:
 * what replay() would launch, without launching it */
static PyObject* hp_splice(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 3 || !PyBytes_Check(args[0]) || !PyList_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "splice(record: bytes, refs: list, n_arrays)");
    return NULL;
  }
  const long n_arrays = PyLong_AsLong(args[2]);
  if (n_arrays == -1 && PyErr_Occurred()) return NULL;
  PyObject* listing = PyList_New(0);
  if (!listing) return NULL;
  PyObject* status = walk_record(args[0], args[1], n_arrays, 0, listing);
  if (!status) {
    Py_DECREF(listing);
    return NULL;
  }
  Py_DECREF(status);
  return listing;
}

/* pool_malloc(pool, size, stream_ident) -> address, or -status on failure */
static PyObject* hp_pool_malloc(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 3) {
    PyErr_SetString(PyExc_TypeError, "pool_malloc takes 3 arguments");
    return NULL;
  }
  uint64_t pool, size, ident, address = 0;
  if (as_u64(args[0], &pool) < 0 || as_u64(args[1], &size) < 0 || as_u64(args[2], &ident) < 0)
    return NULL;
  int status;
  /* the pool may call back into Python (a user's allocator) and may wait for
   * another thread that does: the interpreter lock must not be held */
  Py_BEGIN_ALLOW_THREADS
  status = rt_pool_malloc((void*)(uintptr_t)pool, (size_t)size, ident, &address);
  Py_END_ALLOW_THREADS
  if (status != 0) return PyLong_FromLong(-(long)status);
  return PyLong_FromUnsignedLongLong(address);
}

/* pool_free(pool, address) -> status */
static PyObject* hp_pool_free(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "pool_free takes 2 arguments");
    return NULL;
  }
  uint64_t pool, address;
  if (as_u64(args[0], &pool) < 0 || as_u64(args[1], &address) < 0) return NULL;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = rt_pool_free((void*)(uintptr_t)pool, address);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
}

/* get_device() -> index of the calling thread's current device, or -status */
static PyObject* hp_get_device(PyObject* self, PyObject* unused) {
  (void)self;
  (void)unused;
  int device = 0;
  int status = rt_get_device(&device);
  if (status != 0) return PyLong_FromLong(-(long)status);
  return PyLong_FromLong(device);
}

/* setup(ndarray type, numpy.generic) */
static PyObject* hp_setup(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 2 || !PyType_Check(args[0]) || !PyType_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "setup(array type, numpy.generic)");
    return NULL;
  }
  Py_INCREF(args[0]);
  Py_INCREF(args[1]);
  Py_XDECREF((PyObject*)array_type);
  Py_XDECREF((PyObject*)generic_type);
  array_type = (PyTypeObject*)args[0];
  generic_type = (PyTypeObject*)args[1];
  Py_RETURN_NONE;
}

/* One array's part of a call signature: (dtype, shape, strides, address & 15),
 * or NULL with no error set if the array lives on another device. */
static PyObject* array_signature(PyObject* a, PyObject* dev_id) {
  PyObject *data = NULL, *dev = NULL, *ptr = NULL, *dtype = NULL, *shape = NULL, *strides = NULL;
  PyObject *low = NULL, *out = NULL;
  data = PyObject_GetAttr(a, str_data);
  if (!data) goto done;
  dev = PyObject_GetAttr(data, str_device_id);
  if (!dev) goto done;
  int same = PyObject_RichCompareBool(dev, dev_id, Py_EQ);
  if (same <= 0) goto done;           /* another device (no error) or a failed comparison */
  ptr = PyObject_GetAttr(data, str_ptr);
  if (!ptr) goto done;
  uint64_t address;
  if (as_u64(ptr, &address) < 0) goto done;
  dtype = PyObject_GetAttr(a, str_dtype);
  shape = PyObject_GetAttr(a, str_shape);
  strides = PyObject_GetAttr(a, str_strides);
  low = PyLong_FromLong((long)(address & 15));
  if (!dtype || !shape || !strides || !low) goto done;
  out = PyTuple_Pack(4, dtype, shape, strides, low);
done:
  Py_XDECREF(data);
  Py_XDECREF(dev);
  Py_XDECREF(ptr);
  Py_XDECREF(dtype);
  Py_XDECREF(shape);
  Py_XDECREF(strides);
  Py_XDECREF(low);
  return out;
}

/* The signature of a call's arguments (a tuple or list): device, version, then
 * per argument what launch decisions may depend on: arrays contribute (dtype,
 * shape, strides, alignment of the address), scalars their type.  NULL with no
 * error set when the call must take the full path. */
static PyObject* signature_of(PyObject* call, PyObject* dev_id, PyObject* version) {
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(call);
  PyObject* sig = PyTuple_New(n + 2);
  if (!sig) return NULL;
  Py_INCREF(dev_id);
  PyTuple_SET_ITEM(sig, 0, dev_id);
  Py_INCREF(version);
  PyTuple_SET_ITEM(sig, 1, version);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* a = PySequence_Fast_GET_ITEM(call, i);
    PyTypeObject* t = Py_TYPE(a);
    PyObject* item = NULL;
    if (t == array_type) {
      item = array_signature(a, dev_id);
      if (!item) {
        Py_DECREF(sig);
        return NULL;
      }
    } else if (t == &PyFloat_Type || t == &PyBool_Type || t == &PyComplex_Type) {
      item = (PyObject*)t;
      Py_INCREF(item);
    } else if (t == &PyLong_Type) {
      int overflow = 0;
      (void)PyLong_AsLongLongAndOverflow(a, &overflow);
      if (overflow) {
        Py_DECREF(sig);
        return NULL;
      }
      item = (PyObject*)t;
      Py_INCREF(item);
    } else if (PyType_IsSubtype(t, generic_type)) {
      item = (PyObject*)t;
      Py_INCREF(item);
    } else {
      Py_DECREF(sig);
      return NULL;
    }
    PyTuple_SET_ITEM(sig, i + 2, item);
  }
  return sig;
}

/* signature(args: tuple or list, device id, tuning version) -> tuple, or None when the
 * call must take the full path: everything about the arguments that launch
 * decisions may depend on.  Arrays contribute (dtype, shape, strides,
 * alignment of the address), scalars their type. */
static PyObject* hp_signature(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 3 || !(PyTuple_Check(args[0]) || PyList_Check(args[0]))) {
    PyErr_SetString(PyExc_TypeError, "signature(args: tuple or list, device id, version)");
    return NULL;
  }
  if (!array_type) {
    PyErr_SetString(PyExc_RuntimeError, "signature: setup() has not been called");
    return NULL;
  }
  PyObject* sig = signature_of(args[0], args[1], args[2]);
  if (!sig && !PyErr_Occurred()) Py_RETURN_NONE;
  return sig;
}


/* Whether any pair that `spec` lists of the arrays of `call` (a tuple or list)
 * shares memory; -1 with an error set on failure.  spec: u32 n_arrays, u32
 * n_pairs, per array the lowest and one-past-highest byte it touches relative to
 * its address (i64 each; both 0: it touches nothing), per pair two u32
 * positions; the top bit of the second says that the pair may start at the very
 * same address (the same memory, laid out alike).  Reads addresses only. */
static int overlap_of(PyObject* call, PyObject* spec_bytes) {
  const unsigned char* spec = (const unsigned char*)PyBytes_AS_STRING(spec_bytes);
  const size_t size = (size_t)PyBytes_GET_SIZE(spec_bytes);
  uint32_t n, pairs;
  uint64_t stack_at[64];
  uint64_t* at = stack_at;
  int found = 0;
  if (size < 8) goto malformed;
  memcpy(&n, spec, 4);
  memcpy(&pairs, spec + 4, 4);
  if (size != 8 + 16 * (size_t)n + 8 * (size_t)pairs ||
      (Py_ssize_t)n > PySequence_Fast_GET_SIZE(call))
    goto malformed;
  if (n > 64) {
    at = (uint64_t*)PyMem_Malloc((size_t)n * 8);
    if (!at) {
      PyErr_NoMemory();
      return -1;
    }
  }
  for (uint32_t i = 0; i < n && found == 0; ++i)
    if (address_of(PySequence_Fast_GET_ITEM(call, i), 1, &at[i]) < 0) found = -1;
  for (uint32_t k = 0; k < pairs && found == 0; ++k) {
    uint32_t a, b;
    memcpy(&a, spec + 8 + 16 * (size_t)n + 8 * (size_t)k, 4);
    memcpy(&b, spec + 12 + 16 * (size_t)n + 8 * (size_t)k, 4);
    const int same = b >> 31;
    b &= 0x7fffffffu;
    if (a >= n || b >= n) {
      found = -2;
      break;
    }
    int64_t alo, ahi, blo, bhi;
    memcpy(&alo, spec + 8 + 16 * (size_t)a, 8);
    memcpy(&ahi, spec + 16 + 16 * (size_t)a, 8);
    memcpy(&blo, spec + 8 + 16 * (size_t)b, 8);
    memcpy(&bhi, spec + 16 + 16 * (size_t)b, 8);
    if (alo == ahi || blo == bhi || (same && at[a] == at[b])) continue;
    if (at[a] + (uint64_t)alo < at[b] + (uint64_t)bhi &&
        at[b] + (uint64_t)blo < at[a] + (uint64_t)ahi)
      found = 1;
  }
  if (at != stack_at) PyMem_Free(at);
  if (found != -2) return found;
malformed:
  PyErr_SetString(PyExc_ValueError, "malformed overlap specification");
  return -1;
}

/* overlap(arrays: tuple or list, spec: bytes) -> whether a listed pair shares memory */
static PyObject* hp_overlap(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 2 || !(PyTuple_Check(args[0]) || PyList_Check(args[0])) || !PyBytes_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "overlap(arrays: tuple or list, spec: bytes)");
    return NULL;
  }
  const int found = overlap_of(args[0], args[1]);
  return found < 0 ? NULL : PyBool_FromLong(found);
}

/* call(plans: dict, arrays: list, device id, version, extra: tuple, stream): a recorded call of
 * an operator made again on `arrays`.  `plans` is keyed by the arrays' signature
 * followed by `extra`; a plan is (overlap spec or None, launch record or None,
 * position(s) of the results among the arrays, the recorded call) and, if the
 * launches use temporaries, (a function that allocates, their sizes ...); where
 * the function returns None the plan counts as one without a record.  Returns
 *   None                the call has to be made in full and not to be recorded;
 *   [key]               ... and recorded under `key`;
 *   [key, plan]         the plan has no launch record: the caller replays it;
 *   an int              the status of a launch that failed;
 *   else                the result. */
static PyObject* hp_call(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 6 || !PyDict_Check(args[0]) || !PyList_Check(args[1]) || !PyTuple_Check(args[4])) {
    PyErr_SetString(PyExc_TypeError,
                    "call(plans: dict, arrays: list, device id, version, extra: tuple, stream)");
    return NULL;
  }
  if (!array_type) {
    PyErr_SetString(PyExc_RuntimeError, "call: setup() has not been called");
    return NULL;
  }
  PyObject* arrays = args[1];
  uint64_t stream;
  if (as_u64(args[5], &stream) < 0) return NULL;
  PyObject* sig = signature_of(arrays, args[2], args[3]);
  if (!sig) {
    if (PyErr_Occurred()) return NULL;
    Py_RETURN_NONE;
  }
  PyObject* key = PySequence_Concat(sig, args[4]);
  Py_DECREF(sig);
  if (!key) return NULL;
  PyObject* plan = PyDict_GetItemWithError(args[0], key);
  PyObject* out = NULL;
  if (!plan) {
    if (!PyErr_Occurred()) {
      out = PyList_New(1);
      if (out) PyList_SET_ITEM(out, 0, key);
      else Py_DECREF(key);
    } else {
      Py_DECREF(key);
    }
    return out;
  }
  Py_INCREF(plan);
  PyObject* refs = NULL;                 /* the arrays, then the temporaries */
  const Py_ssize_t parts = PyTuple_Check(plan) ? PyTuple_GET_SIZE(plan) : 0;
  PyObject* temps = parts == 5 ? PyTuple_GET_ITEM(plan, 4) : NULL;
  if (parts < 4 || parts > 5 || (temps && (!PyTuple_Check(temps) || !PyTuple_GET_SIZE(temps)))) {
    PyErr_SetString(PyExc_ValueError, "malformed plan");
    goto done;
  }
  PyObject* spans = PyTuple_GET_ITEM(plan, 0);
  PyObject* record = PyTuple_GET_ITEM(plan, 1);
  PyObject* ret = PyTuple_GET_ITEM(plan, 2);
  if (spans != Py_None) {
    if (!PyBytes_Check(spans)) {
      PyErr_SetString(PyExc_ValueError, "malformed plan");
      goto done;
    }
    const int found = overlap_of(arrays, spans);
    if (found < 0) goto done;
    if (found) {
      out = Py_None;
      Py_INCREF(out);
      goto done;
    }
  }
  int replayed = PyBytes_Check(record);
  const Py_ssize_t n_arrays = PyList_GET_SIZE(arrays);
  if (replayed && temps) {
    refs = PyList_GetSlice(arrays, 0, n_arrays);
    if (!refs) goto done;
    for (Py_ssize_t i = 1; i < PyTuple_GET_SIZE(temps) && replayed; ++i) {
      PyObject* memory = PyObject_CallFunctionObjArgs(PyTuple_GET_ITEM(temps, 0),
                                                      PyTuple_GET_ITEM(temps, i), NULL);
      if (!memory) goto done;
      if (memory == Py_None) replayed = 0;
      const int failed = PyList_Append(refs, memory) < 0;
      Py_DECREF(memory);
      if (failed) goto done;
    }
  }
  if (!replayed) {
    out = PyList_New(2);
    if (out) {
      Py_INCREF(key);
      Py_INCREF(plan);
      PyList_SET_ITEM(out, 0, key);
      PyList_SET_ITEM(out, 1, plan);
    }
    goto done;
  }
  PyObject* launched = walk_record(record, refs ? refs : arrays, (long)n_arrays, stream, NULL);
  if (!launched) goto done;
  if (PyLong_AsLong(launched) != 0) {
    out = launched;
    goto done;
  }
  Py_DECREF(launched);
  /* the results: one position, or a tuple of them */
  const Py_ssize_t count = PyTuple_Check(ret) ? PyTuple_GET_SIZE(ret) : 1;
  PyObject* results = PyTuple_Check(ret) ? PyTuple_New(count) : NULL;
  if (PyTuple_Check(ret) && !results) goto done;
  for (Py_ssize_t i = 0; i < count; ++i) {
    const Py_ssize_t at = PyLong_AsSsize_t(results ? PyTuple_GET_ITEM(ret, i) : ret);
    if (at < 0 || at >= PyList_GET_SIZE(arrays)) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "malformed plan");
      Py_XDECREF(results);
      goto done;
    }
    PyObject* a = PyList_GET_ITEM(arrays, at);
    Py_INCREF(a);
    if (results) PyTuple_SET_ITEM(results, i, a);
    else out = a;
  }
  if (results) out = results;
done:
  Py_XDECREF(refs);
  Py_DECREF(key);
  Py_DECREF(plan);
  return out;
}

/* -- tables of arrays for the kernels that take many arrays in one launch ---------- */

typedef struct {
  uint64_t start, bytes;       /* its memory, for an array stored in one piece */
  uint64_t elements;
  uint32_t type, dense;        /* position in `types`; 1 C order | 2 Fortran order */
  int64_t device;
} Description;

/* The attribute `name` of `a`, looked for among its own attributes `own` before
 * those of its type (145 arrays: 16 us, 18.5 the other way round; lists of
 * hundreds of gradients are described per call). */
static PyObject* attribute(PyObject* a, PyObject* own, PyObject* name) {
  PyObject* v = PyDict_GetItemWithError(own, name);
  if (v) {
    Py_INCREF(v);
    return v;
  }
  return PyErr_Occurred() ? NULL : PyObject_GetAttr(a, name);
}

/* What `a` is; 0, or -1 with an error set.  `item` are the sizes of the types. */
static int describe_one(PyObject* a, PyObject* types, const uint64_t* item, Description* d) {
  if (!array_type || !PyObject_TypeCheck(a, array_type)) {
    PyErr_Format(PyExc_TypeError, "expected cupy.ndarrays, got %.100s", Py_TYPE(a)->tp_name);
    return -1;
  }
  PyObject *data = NULL, *ptr = NULL, *dev = NULL, *size = NULL, *dtype = NULL;
  PyObject *c_order = NULL, *f_order = NULL;
  int rc = -1;
  PyObject* own = PyObject_GenericGetDict(a, NULL);
  if (!own) return -1;
  data = attribute(a, own, str_data);
  if (data) {
    ptr = PyObject_GetAttr(data, str_ptr);
    dev = PyObject_GetAttr(data, str_device_id);
  }
  size = attribute(a, own, str_size);
  dtype = attribute(a, own, str_dtype);
  c_order = attribute(a, own, str_c_contiguous);
  f_order = attribute(a, own, str_f_contiguous);
  Py_DECREF(own);
  if (ptr && dev && size && dtype && c_order && f_order && as_u64(ptr, &d->start) == 0 &&
      as_u64(size, &d->elements) == 0) {
    const Py_ssize_t n_types = PyList_GET_SIZE(types);
    uint32_t type = 0;
    for (; (Py_ssize_t)type < n_types; ++type)
      if (PyObject_RichCompareBool(dtype, PyList_GET_ITEM(types, type), Py_EQ) != 0) break;
    const int c = PyObject_IsTrue(c_order), f = PyObject_IsTrue(f_order);
    d->device = (int64_t)PyLong_AsLongLong(dev);
    if (!PyErr_Occurred()) {
      d->type = type;
      d->dense = (c ? 1u : 0u) | (f ? 2u : 0u);
      d->bytes = (Py_ssize_t)type < n_types ? d->elements * item[type] : 0;
      rc = 0;
    }
  }
  Py_XDECREF(data);
  Py_XDECREF(ptr);
  Py_XDECREF(dev);
  Py_XDECREF(size);
  Py_XDECREF(dtype);
  Py_XDECREF(c_order);
  Py_XDECREF(f_order);
  return rc;
}

#define MAX_TYPES 8

/* The sizes of the elements of `types`; -1 with an error set on failure. */
static int item_sizes(PyObject* types, uint64_t* item) {
  const Py_ssize_t n = PyList_GET_SIZE(types);
  if (n > MAX_TYPES) {
    PyErr_SetString(PyExc_ValueError, "too many types");
    return -1;
  }
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyObject_GetAttr(PyList_GET_ITEM(types, i), str_itemsize);
    const int rc = o ? as_u64(o, &item[i]) : -1;
    Py_XDECREF(o);
    if (rc < 0) return -1;
    if (item[i] == 0 || item[i] > 16) {
      PyErr_SetString(PyExc_ValueError, "unsupported type");
      return -1;
    }
  }
  return 0;
}

static int by_start(const void* a, const void* b) {
  const Description *x = *(const Description* const*)a, *y = *(const Description* const*)b;
  return x->start < y->start ? -1 : x->start > y->start;
}

/* 1 if no two of the n outputs share memory and no input shares memory with an
 * output other than its own, whose very memory it may be.  `sorted`: room for n. */
static int are_apart(const Description* src, const Description* dst, Py_ssize_t n,
                     const Description** sorted) {
  Py_ssize_t m = 0;
  int in_order = 1;                        /* (as arrays cut from one piece are) */
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (!dst[i].bytes) continue;
    if (m && dst[i].start < sorted[m - 1]->start) in_order = 0;
    sorted[m++] = &dst[i];
  }
  if (!in_order) qsort(sorted, (size_t)m, sizeof(*sorted), by_start);
  for (Py_ssize_t k = 1; k < m; ++k)
    if (sorted[k]->start < sorted[k - 1]->start + sorted[k - 1]->bytes) return 0;
  if (src == dst) return 1;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const uint64_t lo = src[i].start, hi = lo + src[i].bytes;
    if (!src[i].bytes || lo == dst[i].start) continue;
    Py_ssize_t a = 0, b = m;               /* the first output that ends behind `lo` */
    while (a < b) {
      const Py_ssize_t mid = (a + b) / 2;
      if (sorted[mid]->start + sorted[mid]->bytes > lo) b = mid;
      else a = mid + 1;
    }
    if (a < m && sorted[a]->start < hi) return 0;
  }
  return 1;
}

typedef struct {
  uint64_t src, dst, n;
  uint32_t first, pad;
} TableEntry;

/* tables(arrays: list, targets: list or None, types: list of dtypes, entries,
 * vectors, device id, write, beside) -> per type met (position of the type, [(table,
 * arrays in it, workgroups)], bytes), or None for arrays that need preparation: of
 * another type or device, not stored in one piece in the order of their targets
 * (None: themselves), of other shapes or types than these, or (with `write`)
 * sharing memory where it is written, with each other, or with the array `beside`
 * (if not None), which is written between the reading of the arrays for their norm
 * and that for their scaling.  A table holds `entries` TableEntry, zeros
 * behind the last; a workgroup takes `vectors` vectors of 16 bytes that start on
 * 16-byte borders of the source.  Empty arrays are left out. */
static PyObject* hp_tables(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 8 || !PyList_Check(args[0]) || !(args[1] == Py_None || PyList_Check(args[1])) ||
      !PyList_Check(args[2])) {
    PyErr_SetString(PyExc_TypeError,
                    "tables(arrays: list, targets: list or None, types: list, entries, vectors, "
                    "device id, write, beside)");
    return NULL;
  }
  uint64_t item[MAX_TYPES], entries, vectors;
  if (item_sizes(args[2], item) < 0) return NULL;
  if (as_u64(args[3], &entries) < 0 || as_u64(args[4], &vectors) < 0) return NULL;
  const long long device = PyLong_AsLongLong(args[5]);
  if (device == -1 && PyErr_Occurred()) return NULL;
  const int write = PyObject_IsTrue(args[6]);
  if (write < 0) return NULL;
  if (entries == 0 || entries > 4096 || vectors == 0 || vectors > (1u << 24)) {
    PyErr_SetString(PyExc_ValueError, "tables: entries or vectors out of range");
    return NULL;
  }
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  const Py_ssize_t n_types = PyList_GET_SIZE(args[2]);
  const int own = args[1] == Py_None;
  if (!own && PyList_GET_SIZE(args[1]) != n) {
    PyErr_SetString(PyExc_ValueError, "tables: as many targets as arrays are expected");
    return NULL;
  }
  PyObject* result = NULL;
  TableEntry* table = NULL;
  Description* src = PyMem_New(Description, (size_t)(2 * n + 1));
  const Description** sorted = PyMem_New(const Description*, (size_t)(n + 1));
  Description* dst = own || !src ? src : src + n;
  if (!src || !sorted) {
    PyErr_NoMemory();
    goto done;
  }
  int plain = 1;
  for (Py_ssize_t i = 0; i < n && plain; ++i) {
    if (i >= PyList_GET_SIZE(args[0]) || (!own && i >= PyList_GET_SIZE(args[1]))) {
      PyErr_SetString(PyExc_RuntimeError, "tables: a list changed on the way");
      goto done;
    }
    PyObject* a = PyList_GET_ITEM(args[0], i);
    if (describe_one(a, args[2], item, &src[i]) < 0) goto done;
    if (!own) {
      PyObject* b = PyList_GET_ITEM(args[1], i);
      if (describe_one(b, args[2], item, &dst[i]) < 0) goto done;
      PyObject* sa = PyObject_GetAttr(a, str_shape);
      PyObject* sb = sa ? PyObject_GetAttr(b, str_shape) : NULL;
      const int same = sb ? PyObject_RichCompareBool(sa, sb, Py_EQ) : -1;
      Py_XDECREF(sa);
      Py_XDECREF(sb);
      if (same < 0) goto done;
      if (!same || src[i].type != dst[i].type || dst[i].device != device) plain = 0;
    }
    if ((Py_ssize_t)src[i].type >= n_types || src[i].device != device ||
        !(src[i].dense & dst[i].dense))
      plain = 0;
  }
  if (plain && write && args[7] != Py_None) {
    Description one;
    if (describe_one(args[7], args[2], item, &one) < 0) goto done;
    /* (a type that is not listed: as if it were one of 16 bytes) */
    const uint64_t bytes = one.bytes ? one.bytes : one.elements * 16;
    if (!one.dense) plain = 0;
    for (Py_ssize_t i = 0; i < n; ++i)
      if ((dst[i].start < one.start + bytes && one.start < dst[i].start + dst[i].bytes) ||
          (src[i].start < one.start + bytes && one.start < src[i].start + src[i].bytes))
        plain = 0;
  }
  if (!plain || (write && !are_apart(src, dst, n, sorted))) {
    result = Py_None;
    Py_INCREF(result);
    goto done;
  }
  table = PyMem_New(TableEntry, (size_t)entries);
  if (!table) {
    PyErr_NoMemory();
    goto done;
  }
  result = PyList_New(0);
  for (Py_ssize_t t = 0; result && t < n_types; ++t) {
    PyObject* launches = NULL;           /* (empty where all arrays of a type are) */
    uint64_t used = 0, blocks = 0, bytes = 0;
    int failed = 0;
    for (Py_ssize_t i = 0; i <= n && !failed; ++i) {
      const int last = i == n;
      if (!last && (Py_ssize_t)src[i].type != t) continue;
      if (!last && !launches && !(launches = PyList_New(0))) {
        failed = 1;
        break;
      }
      if (!last && src[i].elements == 0) continue;
      if (used && (last || used == entries)) {
        /* (the kernels count workgroups of 256 threads in 32 bits) */
        if (blocks > 0xffffffffull / 256) {
          PyErr_SetString(PyExc_ValueError, "more than 2**39 bytes of arrays in one launch");
          failed = 1;
          break;
        }
        memset(table + used, 0, (size_t)(entries - used) * sizeof(TableEntry));
        PyObject* one = Py_BuildValue("y#KK", (const char*)table,
                                      (Py_ssize_t)(entries * sizeof(TableEntry)),
                                      (unsigned long long)used, (unsigned long long)blocks);
        if (!one || PyList_Append(launches, one) < 0) failed = 1;
        Py_XDECREF(one);
        used = blocks = 0;
      }
      if (last || failed) break;
      const uint64_t per = 16 / item[t] * vectors;
      const uint64_t count = ((src[i].start & 15) / item[t] + src[i].elements + per - 1) / per;
      TableEntry* e = &table[used++];
      e->src = src[i].start;
      e->dst = dst[i].start;
      e->n = src[i].elements;
      e->first = (uint32_t)blocks;
      e->pad = 0;
      blocks += count;
      bytes += src[i].bytes;
    }
    if (!failed && launches) {
      PyObject* one = Py_BuildValue("nOK", t, launches, (unsigned long long)bytes);
      if (!one || PyList_Append(result, one) < 0) failed = 1;
      Py_XDECREF(one);
    }
    Py_XDECREF(launches);
    if (failed) Py_CLEAR(result);
  }
done:
  PyMem_Free(table);
  PyMem_Free((void*)sorted);
  PyMem_Free(src);
  return result;
}

/* describe(arrays: list, types: list of dtypes) -> bytes, per array: u64 address,
 * u64 elements, u32 position of its dtype in `types` (their number: none of
 * them), u32 1 if stored in C order | 2 if in Fortran order, i64 device. */
static PyObject* hp_describe(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 2 || !PyList_Check(args[0]) || !PyList_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "describe(arrays: list, types: list)");
    return NULL;
  }
  uint64_t item[MAX_TYPES];
  if (item_sizes(args[1], item) < 0) return NULL;
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  PyObject* out = PyBytes_FromStringAndSize(NULL, n * 32);
  if (!out) return NULL;
  unsigned char* to = (unsigned char*)PyBytes_AS_STRING(out);
  memset(to, 0, (size_t)n * 32);
  for (Py_ssize_t i = 0; i < n && i < PyList_GET_SIZE(args[0]); ++i, to += 32) {
    Description d;
    if (describe_one(PyList_GET_ITEM(args[0], i), args[1], item, &d) < 0) {
      Py_DECREF(out);
      return NULL;
    }
    memcpy(to, &d.start, 8);
    memcpy(to + 8, &d.elements, 8);
    memcpy(to + 16, &d.type, 4);
    memcpy(to + 20, &d.dense, 4);
    memcpy(to + 24, &d.device, 8);
  }
  return out;
}

static PyMethodDef methods[] = {
    {"call", (PyCFunction)(void (*)(void))hp_call, METH_FASTCALL,
     "call(plans, arrays, device id, version, extra, stream) -> result of a recorded call made again"},
    {"tables", (PyCFunction)(void (*)(void))hp_tables, METH_FASTCALL,
     "tables(arrays, targets, types, entries, vectors, device id, write, beside) -> tables or None"},
    {"describe", (PyCFunction)(void (*)(void))hp_describe, METH_FASTCALL,
     "describe(arrays, types) -> addresses, sizes, types and layouts as bytes"},
    {"overlap", (PyCFunction)(void (*)(void))hp_overlap, METH_FASTCALL,
     "overlap(arrays, spec) -> whether a listed pair of arrays shares memory"},
    {"get_device", hp_get_device, METH_NOARGS, "get_device() -> device index or -status"},
    {"setup", (PyCFunction)(void (*)(void))hp_setup, METH_FASTCALL,
     "setup(array type, numpy.generic)"},
    {"signature", (PyCFunction)(void (*)(void))hp_signature, METH_FASTCALL,
     "signature(args, device id, version) -> tuple or None"},
    {"launch", (PyCFunction)(void (*)(void))hp_launch, METH_FASTCALL,
     "launch(function, gx, gy, gz, bx, by, bz, shared_mem, stream, arg_block) -> status"},
    {"replay", (PyCFunction)(void (*)(void))hp_replay, METH_FASTCALL,
     "replay(record, refs, n_arrays, stream) -> status"},
    {"splice", (PyCFunction)(void (*)(void))hp_splice, METH_FASTCALL,
     "splice(record, refs, n_arrays) -> list of launches as replay() would make them"},
    {"pool_malloc", (PyCFunction)(void (*)(void))hp_pool_malloc, METH_FASTCALL,
     "pool_malloc(pool, size, stream_ident) -> address or -status"},
    {"pool_free", (PyCFunction)(void (*)(void))hp_pool_free, METH_FASTCALL,
     "pool_free(pool, address) -> status"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hotpath",
                                    "Per-launch host calls of cupy_amd in C.", -1, methods,
                                    NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__hotpath(void) {
  str_data = PyUnicode_InternFromString("data");
  str_ptr = PyUnicode_InternFromString("ptr");
  str_dtype = PyUnicode_InternFromString("dtype");
  str_shape = PyUnicode_InternFromString("_shape");
  str_strides = PyUnicode_InternFromString("_strides");
  str_device_id = PyUnicode_InternFromString("device_id");
  str_size = PyUnicode_InternFromString("size");
  str_itemsize = PyUnicode_InternFromString("itemsize");
  str_c_contiguous = PyUnicode_InternFromString("_c_contiguous");
  str_f_contiguous = PyUnicode_InternFromString("_f_contiguous");
  if (!str_data || !str_ptr || !str_dtype || !str_shape || !str_strides || !str_device_id ||
      !str_size || !str_itemsize || !str_c_contiguous || !str_f_contiguous)
    return NULL;
  return PyModule_Create(&module);
}
