// Where the memory of many torch tensors lies and what it holds, in one call from Python: torch's own attributes cost some 40 ns
// each, and an optimizer step over 150 tensors asks for a thousand of them.  (Host code: compiled by g++ against torch's headers.)
#include <torch/extension.h>
#include <cstdint>
#include <vector>

namespace {

struct Layout {
  uint64_t address;
  int64_t elements;
  int64_t kind;            // scalar type, + 256: contiguous; -1: no tensor
};

// bytes: a Layout for each entry, a tensor or None.  Equal bytes: the same memory is taken for the same values.
py::bytes layout(const py::list& tensors) {
  std::vector<Layout> out;
  out.reserve(tensors.size());
  for (const py::handle& h : tensors) {
    if (h.is_none()) {
      out.push_back({0, 0, -1});
      continue;
    }
    if (!THPVariable_Check(h.ptr())) throw py::type_error("a tensor or None is required");
    const at::Tensor& t = THPVariable_Unpack(h.ptr());
    out.push_back({(uint64_t)(uintptr_t)t.data_ptr(), t.numel(), (int64_t)t.scalar_type() + (t.is_contiguous() ? 256 : 0)});
  }
  return py::bytes((const char*)out.data(), out.size() * sizeof(Layout));
}

}  // namespace

PYBIND11_MODULE(_layout, m) { m.def("layout", &layout); }
