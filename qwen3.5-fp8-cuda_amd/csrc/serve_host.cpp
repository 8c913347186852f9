// The host side of a serving step's calls (tables.py): checks the torch tensors of a call and
// launches it.  Each function takes the address of the C entry point and the call's tensors; it
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
      Py_BEGIN_ALLOW_THREADS
      rc = entry(pages, (int)n, (int)max_pages, page_size, length, fresh, done, free_pages, (int)n_pages, n_free, length_out,
                 n_free_out, at, seq, (int)T, start, last, stream);
      Py_END_ALLOW_THREADS
    }
    return status(a.good, rc);
  });
}

PyMethodDef methods[] = {
    {"step", (PyCFunction)(void (*)(void))step_tables, METH_FASTCALL, "Check the tensors of PageTables.step and launch it."},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serve_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__serve_host() { return PyModule_Create(&module); }
