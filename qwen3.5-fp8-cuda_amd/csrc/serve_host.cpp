// The host side of a serving step's calls (tables.py, adapters.py, sampling.py): checks the torch tensors of
// a call and launches it.  Each function takes the address of the C entry point and the call's tensors; it
// returns the entry point's status, or None where a tensor is not what the call takes: the
// Python caller then finds out which, for the message.
#include "host_args.h"

#include "../../include/qwen35_fp8_hip.h"

namespace {

// step(entry, device, pages, page_size, length, new, done, free, n_free, length_out, n_free_out,
//      at, seq, start, last, stream)
PyObject* step_tables(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  if (!takes(nargs, 16)) return nullptr;
  return guarded([&]() -> PyObject* {
    Args a{v};
    const auto entry = a.address<decltype(&qh_page_tables_step)>(0);
    a.dev = (int)PyLong_AsLong(v[1]);
    const int page_size = (int)PyLong_AsLong(v[3]);
    void* stream = a.address<void*>(15);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor* table = a.tensor(2, at::kInt, 2);
    int* pages = (int*)a.dense(2, at::kInt, {-1, -1});
    const int64_t n = table ? table->size(0) : 0, max_pages = table ? table->size(1) : 0;
    const int* length = (const int*)a.dense(4, at::kInt, {n});
    const int* fresh = (const int*)a.dense(5, at::kInt, {n});
    const int* done = (const int*)a.dense_or_none(6, at::kInt, {n});
    const at::Tensor* pool = a.tensor(7, at::kInt, 1);
    int* free_pages = (int*)a.dense(7, at::kInt, {-1});
    const int* n_free = (const int*)a.dense(8, at::kInt, {1});
    int* length_out = (int*)a.dense(9, at::kInt, {n});
    int* n_free_out = (int*)a.dense(10, at::kInt, {1});
    const at::Tensor* where = a.tensor(11, at::kInt, 1);
    const int64_t T = where ? where->size(0) : 0;
    const bool flat = v[12] != Py_None;
    int* at = (int*)a.dense(11, at::kInt, {flat ? T : n});
    int* seq = (int*)a.dense_or_none(12, at::kInt, {T});
    int* start = (int*)a.dense_or_none(13, at::kInt, {n + 1});
    int* last = (int*)a.dense_or_none(14, at::kInt, {n});
    a.good = a.good && flat == (v[13] != Py_None);
    int rc = 0;
    const int64_t n_pages = pool ? pool->size(0) : 0;
    a.good = a.good && is_int(n) && is_int(max_pages) && is_int(n_pages) && is_int(T);
    if (a.good) {
      if (flat && T == 0) seq = start;  // an empty tensor's address is null, which would say: one token a row
      Py_BEGIN_ALLOW_THREADS
      rc = entry(pages, (int)n, (int)max_pages, page_size, length, fresh, done, free_pages, (int)n_pages, n_free, length_out,
                 n_free_out, at, seq, (int)T, start, last, stream);
      Py_END_ALLOW_THREADS
    }
    return status(a.good, rc);
  });
}

// add(entry, device, a, b, scale, x, ids, y, ws, out, stream)
PyObject* add_adapters(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  if (!takes(nargs, 11)) return nullptr;
  return guarded([&]() -> PyObject* {
    Args args{v};
    const auto entry = args.address<decltype(&qh_adapters_add)>(0);
    args.dev = (int)PyLong_AsLong(v[1]);
    void* stream = args.address<void*>(10);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor* at = args.tensor(2, at::kBFloat16, 3);
    const int64_t n = at ? at->size(0) : 0, R = at ? at->size(1) : 0, K = at ? at->size(2) : 0;
    const void* a = args.dense(2, at::kBFloat16, {-1, -1, -1});
    const at::Tensor* bt = args.tensor(3, at::kBFloat16, 3);
    const int64_t N = bt ? bt->size(1) : 0;
    const void* b = args.dense(3, at::kBFloat16, {n, N, R});
    const float* scale = (const float*)args.dense(4, at::kFloat, {n});
    const at::Tensor* x = args.matrix(5, -1, K);
    const int64_t T = x ? x->size(0) : 0;
    const int* ids = (const int*)args.dense(6, at::kInt, {T});
    const at::Tensor* y = args.matrix(7, T, N);
    void* ws = args.dense(8, at::kByte, {-1});
    const at::Tensor* out = args.matrix(9, T, N);
    int rc = 0;
    args.good = args.good && is_int(n) && is_int(R) && is_int(K) && is_int(N) && is_int(T);
    if (args.good) {
      const void *xp = x->data_ptr(), *yp = y->data_ptr();
      void* op = out->data_ptr();
      const int64_t xs = step(*x, 0), ys = step(*y, 0), os = step(*out, 0);
      const size_t ws_bytes = (size_t)THPVariable_Unpack(v[8]).size(0);
      Py_BEGIN_ALLOW_THREADS
      rc = entry(a, b, scale, (int)n, (int)R, (int)K, (int)N, xp, xs, ids, (int)T, yp, ys, op, os, ws, ws_bytes, stream);
      Py_END_ALLOW_THREADS
    }
    return status(args.good, rc);
  });
}

// sample(entry, device, logits, u, ws, temperature, top_k, top_p, min_p, out, logprob, stream)
PyObject* sample_rows(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  if (!takes(nargs, 12)) return nullptr;
  return guarded([&]() -> PyObject* {
    Args a{v};
    const auto entry = a.address<decltype(&qh_sample_rows)>(0);
    a.dev = (int)PyLong_AsLong(v[1]);
    void* stream = a.address<void*>(11);
    if (PyErr_Occurred()) return nullptr;
    const bool f32 = THPVariable_Check(v[2]) && THPVariable_Unpack(v[2]).scalar_type() == at::kFloat;
    const at::Tensor* x = a.matrix(2, -1, -1, f32 ? at::kFloat : at::kBFloat16);
    const int64_t B = x ? x->size(0) : 0, V = x ? x->size(1) : 0;
    const float* u = (const float*)a.dense(3, at::kFloat, {B});
    void* ws = a.dense(4, at::kByte, {-1});
    const float* heat = (const float*)a.dense_or_none(5, at::kFloat, {B});
    const int* top_k = (const int*)a.dense_or_none(6, at::kInt, {B});
    const float* top_p = (const float*)a.dense_or_none(7, at::kFloat, {B});
    const float* min_p = (const float*)a.dense_or_none(8, at::kFloat, {B});
    int64_t* token = (int64_t*)a.dense(9, at::kLong, {B});
    float* logprob = (float*)a.dense_or_none(10, at::kFloat, {B});
    int rc = 0;
    a.good = a.good && is_int(B) && is_int(V);
    if (a.good) {
      const void* xp = x->data_ptr();
      const int64_t stride = step(*x, 0);
      const size_t ws_bytes = (size_t)THPVariable_Unpack(v[4]).size(0);
      Py_BEGIN_ALLOW_THREADS
      rc = entry(xp, stride, f32, (int)B, (int)V, u, heat, top_k, top_p, min_p, token, logprob, ws, ws_bytes, stream);
      Py_END_ALLOW_THREADS
    }
    return status(a.good, rc);
  });
}

PyMethodDef methods[] = {
    {"sample", (PyCFunction)(void (*)(void))sample_rows, METH_FASTCALL, "Check the tensors of sampling.sample and launch it."},
    {"add", (PyCFunction)(void (*)(void))add_adapters, METH_FASTCALL, "Check the tensors of Adapters.add and launch it."},
    {"step", (PyCFunction)(void (*)(void))step_tables, METH_FASTCALL, "Check the tensors of PageTables.step and launch it."},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serve_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__serve_host() { return PyModule_Create(&module); }
