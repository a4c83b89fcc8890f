// What the calls on torch tensors share: checks of arguments, results, the stream, and what a captured backward pass
// has to be told.
#ifndef AMSIM_TORCH_H_
#define AMSIM_TORCH_H_

#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "amsim.h"

namespace amsim_torch {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---- arguments --------------------------------------------------------------------------------------------------

[[noreturn]] inline void value_error(const std::string &what) { throw py::value_error(what); }
[[noreturn]] inline void type_error(const std::string &what) { throw py::type_error(what); }

inline int code_of(at::ScalarType t)
{
    return t == at::kFloat ? AMSIM_DTYPE_F32 : t == at::kBFloat16 ? AMSIM_DTYPE_BF16 : t == at::kHalf ? AMSIM_DTYPE_F16 : -1;
}
inline std::string name_of(at::ScalarType t) { return py::str(py::reinterpret_borrow<py::object>((PyObject *)torch::getTHPDtype(t))); }
inline int known(at::ScalarType t, const char *name)
{
    const int code = code_of(t);
    if (code < 0) type_error(std::string(name) + " must be float32, bfloat16 or float16, got " + name_of(t));
    return code;
}
inline int result_code(py::handle dtype, at::ScalarType &t)
{
    if (THPDtype_Check(dtype.ptr())) {
        t = ((THPDtype *)dtype.ptr())->scalar_type;
        const int code = code_of(t);
        if (code >= 0) return code;
    }
    type_error("the result's type must be float32, bfloat16 or float16, got " + std::string(py::str(dtype)));
}

// the library launches on the current device
inline const Tensor &on_device(const Tensor &t, const char *name)
{
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided) type_error(std::string(name) + " must be a tensor in device memory (there is no CPU path)");
    if (t.get_device() != c10::hip::current_device())
        value_error(std::string(name) + " is on device " + std::to_string(t.get_device()) + ", which is not the current one");
    return t;
}
inline const Tensor &tensor(py::handle h, const char *name)
{
    if (!THPVariable_Check(h.ptr())) type_error(std::string(name) + " must be a tensor in device memory (there is no CPU path)");
    return THPVariable_Unpack(h.ptr());
}
inline std::optional<Tensor> maybe_tensor(py::handle h, const char *name)
{
    if (h.is_none()) return std::nullopt;
    return tensor(h, name);
}

// for calls that are no part of a graph: what would need a derivative is refused, and not cut off without a word
inline void no_derivative(const Tensor &t, const char *name, const char *call, const char *train)
{
    if (at::GradMode::is_enabled() && t.requires_grad())
        throw std::runtime_error(std::string(call) + " has no gradient and " + name + " requires one: train through " + train + ", or call it under torch.no_grad()");
    if (t._fw_grad(0).defined()) type_error(std::string(call) + " has no forward-mode derivative");
}

inline void *stream() { return c10::hip::getCurrentHIPStream().stream(); }

inline void check(int status)
{
    if (status != 0) py::module_::import("approxtrain_amd._lib").attr("check")(status);
}

inline Tensor bytes(int64_t n, const Tensor &like) { return at::empty({n}, like.options().dtype(at::kByte)); }
inline Tensor matrix(int64_t rows, int64_t cols, const Tensor &like, at::ScalarType t) { return at::empty({rows, cols}, like.options().dtype(t)); }

// A matrix as the library reads it, in place where either of its axes is contiguous: its transpose if `swapped`.
struct Source {
    Tensor t;
    int dtype;
    int64_t rows, cols, stride;
    bool swapped;
};
inline Source source(const Tensor &given, const char *name)
{
    Source s{on_device(given, name), known(given.scalar_type(), name), 0, 0, 0, false};
    if (given.dim() != 2) value_error(std::string(name) + " must be a matrix");
    s.rows = given.size(0), s.cols = given.size(1);
    if (s.rows == 0 || s.cols == 0) value_error(std::string(name) + " is empty: blocks of no elements have no scale");
    if (s.t.is_neg()) s.t = s.t.resolve_neg();
    if (s.t._is_zerotensor()) s.t = at::zeros(s.t.sizes(), s.t.options());  // (zeros that take no memory)
    const int64_t s0 = s.t.stride(0), s1 = s.t.stride(1);
    if ((s1 == 1 || s.cols == 1) && (s0 >= s.cols || s.rows == 1)) {
        s.stride = s.rows > 1 ? s0 : s.cols;
    } else if ((s0 == 1 || s.rows == 1) && (s1 >= s.rows || s.cols == 1)) {
        s.stride = s.cols > 1 ? s1 : s.rows;
        std::swap(s.rows, s.cols);
        s.swapped = true;
    } else {
        s.t = s.t.contiguous();
        s.stride = s.cols;
    }
    return s;
}
// ... with its rows contiguous
inline Source row_source(const Tensor &given, const char *name)
{
    Source s = source(given, name);
    if (s.swapped) {
        s.t = s.t.contiguous();
        std::swap(s.rows, s.cols);
        s.stride = s.cols;
        s.swapped = false;
    }
    return s;
}

struct Bias {
    std::optional<Tensor> t;
    int dtype = 0;
    const void *ptr() const { return t ? t->data_ptr() : nullptr; }
};
inline Bias bias_of(const std::optional<Tensor> &b, int64_t units, const Tensor &like)
{
    if (!b) return {};
    on_device(*b, "bias");
    if (b->get_device() != like.get_device()) value_error("bias must be on the operands' device");
    const int dtype = known(b->scalar_type(), "bias");
    if (b->dim() != 1 || b->size(0) != units) value_error("bias must have one entry per output channel");
    return {b->_is_zerotensor() ? at::zeros(b->sizes(), b->options()) : b->contiguous().resolve_neg(), dtype};
}

// ---- backward passes ---------------------------------------------------------------------------------------------

// A leaf has one node that adds its gradients, on the stream that it was made on, for as long as a graph of it lives.  Where
// that is the default stream, a captured backward pass would have to wait for a captured event there, which cannot be
// recorded and ends the process in the engine's thread: seen here first, it is an error like others.
inline bool adds_on_default_stream(const Tensor &t)
{
    const auto node = t.requires_grad() && t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : nullptr;
    const auto stream = node ? node->stream() : std::nullopt;
    return stream && stream->id() == 0;
}
inline bool capturing()
{
    const auto current = c10::hip::getCurrentHIPStream();
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    return current.id() != 0 && hipStreamIsCapturing(current.stream(), &status) == hipSuccess && status != hipStreamCaptureStatusNone;
}

// Gradients of gradients are not provided: in a backward pass that is recorded `grads` stay usable, and asking for theirs
// is an error that says so.
inline void no_second_derivative(variable_list &grads, bool asked, const std::string &call)
{
    if (!at::GradMode::is_enabled() || !asked) return;
    variable_list some;
    for (const Tensor &g : grads)
        if (g.defined()) some.push_back(g.detach().set_requires_grad(true));
    const auto error = std::make_shared<torch::autograd::DelayedError>("gradients of " + call + "'s gradients are not provided", (int64_t)some.size());
    some = (*error)(std::move(some));
    size_t j = 0;
    for (Tensor &g : grads)
        if (g.defined()) g = some[j++];
}

// the calls of amsim_torch_rows.cc and amsim_torch_i8.cc
void bind_rows(py::module_ &m);
void bind_i8(py::module_ &m);

}  // namespace amsim_torch
#endif  // AMSIM_TORCH_H_
