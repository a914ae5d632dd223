// fgt_native.cpp — the Python extension `fugatensor_b200._native`: prepared
// programs of the C ABI (include/fgt.h) for the engine's cache-hit dispatch.
//
// Shape of the reference's native session API for this path:
// Session.prepare_program(..., graph) returns a PreparedProgram whose run
// enqueues the whole plan, replayed as one CUDA graph
// (cpp/ask_runtime.cpp:789-843; Python side src/fugatensor/_ask/executable.py:120-152),
// and the cache-hit dispatch calls it natively (cpp/lazy.cpp:946-948).
// Here prepare_program(spec_handle, graph) wraps fgt_program_create and
// Program.run wraps fgt_program_run with the GIL released; buffers cross as
// integer device addresses. Statuses are returned as integers (the Python
// layer reads fgt_last_error() on the same thread and raises).
// The vocabulary operators (fgt_embedding, fgt_cross_entropy,
// fgt_adjust_logits) cross the same way: descriptor fields, then addresses.
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <vector>

#include "fgt.h"

namespace py = pybind11;

namespace {

class Program {
 public:
  Program(uintptr_t spec, bool graph) {
    const fgt_status st = fgt_program_create(reinterpret_cast<const fgt_spec*>(spec), graph ? 1 : 0, &p_);
    if (st != FGT_OK) throw std::runtime_error(std::string("fgt_program_create: ") + fgt_last_error());
    graph_ = graph;
  }
  ~Program() { fgt_program_destroy(p_); }
  Program(const Program&) = delete;
  Program& operator=(const Program&) = delete;

  int run(const std::vector<uintptr_t>& inputs, const std::vector<uintptr_t>& outputs, uintptr_t workspace,
          size_t workspace_bytes, uintptr_t stream) {
    fgt_status st;
    {
      py::gil_scoped_release release;
      st = fgt_program_run(p_, reinterpret_cast<const void* const*>(inputs.data()),
                           reinterpret_cast<void* const*>(outputs.data()), reinterpret_cast<void*>(workspace),
                           workspace_bytes, reinterpret_cast<void*>(stream));
    }
    return (int)st;
  }
  int kernel_count() const { return fgt_program_kernel_count(p_); }
  bool graph() const { return graph_; }

 private:
  fgt_program* p_ = nullptr;
  bool graph_ = true;
};

fgt_embedding_desc embedding_desc(int dtype, int index_dtype, int64_t vocab, int64_t dim, int64_t count, float scale,
                                  int64_t padding) {
  fgt_embedding_desc d{};
  d.dtype = dtype;
  d.index_dtype = index_dtype;
  d.vocab = vocab;
  d.dim = dim;
  d.count = count;
  d.padding_index = padding;
  d.scale = scale;
  return d;
}

fgt_cross_entropy_desc loss_desc(int dtype, int target_dtype, int reduction, float smoothing, float z, float grad_scale,
                                 int64_t rows, int64_t vocab, int64_t ignore) {
  fgt_cross_entropy_desc d{};
  d.dtype = dtype;
  d.target_dtype = target_dtype;
  d.reduction = reduction;
  d.label_smoothing = smoothing;
  d.z_loss = z;
  d.grad_scale = grad_scale;
  d.rows = rows;
  d.vocab = vocab;
  d.ignore_index = ignore;
  return d;
}

template <class T> T* at(uintptr_t p) { return reinterpret_cast<T*>(p); }

template <class D> size_t workspace_bytes(fgt_status (*query)(const D*, size_t*), const D& d) {
  size_t n = 0;
  if (query(&d, &n) != FGT_OK) throw std::runtime_error(fgt_last_error());
  return n;
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.doc() = "prepared programs of the fgt C ABI (CUDA graph replay of a partition's kernels)";
  m.def("abi_version", &fgt_abi_version);
  py::class_<Program>(m, "Program")
      .def_property_readonly("kernel_count", &Program::kernel_count)
      .def_property_readonly("graph", &Program::graph)
      .def("run", &Program::run, py::arg("inputs"), py::arg("outputs"), py::arg("workspace"),
           py::arg("workspace_bytes"), py::arg("stream"));
  m.def(
      "prepare_program",
      [](uintptr_t spec, bool graph) { return new Program(spec, graph); }, py::arg("spec"), py::arg("graph") = true,
      py::return_value_policy::take_ownership);
  m.def("embedding", [](int dtype, int index_dtype, int64_t vocab, int64_t dim, int64_t count, float scale,
                        uintptr_t table, uintptr_t indices, uintptr_t out, uintptr_t stream) {
    const fgt_embedding_desc d = embedding_desc(dtype, index_dtype, vocab, dim, count, scale, -1);
    return (int)fgt_embedding(&d, at<void>(table), at<void>(indices), at<void>(out), at<void>(stream));
  });
  m.def("embedding_grad_workspace", [](int dtype, int index_dtype, int64_t vocab, int64_t dim, int64_t count,
                                       float scale, int64_t padding) {
    const fgt_embedding_desc d = embedding_desc(dtype, index_dtype, vocab, dim, count, scale, padding);
    return workspace_bytes(&fgt_embedding_grad_workspace, d);
  });
  m.def("embedding_grad", [](int dtype, int index_dtype, int64_t vocab, int64_t dim, int64_t count, float scale,
                             int64_t padding, uintptr_t indices, uintptr_t dy, uintptr_t dtable, uintptr_t workspace,
                             size_t bytes, uintptr_t stream) {
    const fgt_embedding_desc d = embedding_desc(dtype, index_dtype, vocab, dim, count, scale, padding);
    return (int)fgt_embedding_grad(&d, at<void>(indices), at<void>(dy), at<void>(dtable), at<void>(workspace), bytes,
                                   at<void>(stream));
  });
  m.def("cross_entropy_workspace", [](int dtype, int target_dtype, int reduction, float smoothing, float z,
                                      float grad_scale, int64_t rows, int64_t vocab, int64_t ignore) {
    const fgt_cross_entropy_desc d =
        loss_desc(dtype, target_dtype, reduction, smoothing, z, grad_scale, rows, vocab, ignore);
    return workspace_bytes(&fgt_cross_entropy_workspace, d);
  });
  m.def("cross_entropy", [](int dtype, int target_dtype, int reduction, float smoothing, float z, float grad_scale,
                            int64_t rows, int64_t vocab, int64_t ignore, uintptr_t logits, uintptr_t targets,
                            uintptr_t seed, uintptr_t loss, uintptr_t dlogits, uintptr_t workspace, size_t bytes,
                            uintptr_t stream) {
    const fgt_cross_entropy_desc d =
        loss_desc(dtype, target_dtype, reduction, smoothing, z, grad_scale, rows, vocab, ignore);
    return (int)fgt_cross_entropy(&d, at<void>(logits), at<void>(targets), at<float>(seed), at<float>(loss),
                                  at<void>(dlogits), at<void>(workspace), bytes, at<void>(stream));
  });
  m.def("adjust_logits", [](int dtype, int token_dtype, int length_dtype, int bias_dtype, int64_t rows, int64_t vocab,
                            int64_t history, int64_t biases, float repetition, float presence, float frequency,
                            uintptr_t logits, uintptr_t tokens, uintptr_t lengths, uintptr_t prompt_lengths,
                            uintptr_t repetitions, uintptr_t presences, uintptr_t frequencies, uintptr_t bias_tokens,
                            uintptr_t bias, uintptr_t allowed, uintptr_t out, uintptr_t stream) {
    fgt_adjust_logits_desc d{};
    d.dtype = dtype;
    d.token_dtype = token_dtype;
    d.length_dtype = length_dtype;
    d.bias_dtype = bias_dtype;
    d.rows = rows;
    d.vocab = vocab;
    d.history = history;
    d.biases = biases;
    d.repetition = repetition;
    d.presence = presence;
    d.frequency = frequency;
    fgt_adjust_logits_buffers b{};
    b.logits = at<void>(logits);
    b.tokens = at<void>(tokens);
    b.lengths = at<void>(lengths);
    b.prompt_lengths = at<void>(prompt_lengths);
    b.repetition = at<float>(repetitions);
    b.presence = at<float>(presences);
    b.frequency = at<float>(frequencies);
    b.bias_tokens = at<void>(bias_tokens);
    b.bias = at<float>(bias);
    b.allowed = at<uint32_t>(allowed);
    b.out = at<void>(out);
    return (int)fgt_adjust_logits(&d, &b, at<void>(stream));
  });
}
