// The products in 8-bit integers on torch tensors: arguments, results, workspaces, the stream and the training layer's node
// of the autograd graph on top of the C ABI (as amsim_torch.cc for the 4-bit products).
#include "amsim_torch.h"

using namespace amsim_torch;

namespace {

int64_t operand_bytes(int64_t rows, int64_t length)
{
    const size_t n = amsim_i8_operand_workspace_bytes(rows, length);
    if (n == 0) value_error("a " + std::to_string(rows) + " x " + std::to_string(length) + " tensor is out of the 8-bit products' range");
    return (int64_t)n;
}
// the bytes of an I8Tensor
const Tensor &operand(const Tensor &data, int64_t rows, int64_t length, const char *name)
{
    on_device(data, name);
    if (data.scalar_type() != at::kByte || !data.is_contiguous() || data.numel() != operand_bytes(rows, length))
        value_error(std::string(name) + "'s data are not those of a " + std::to_string(rows) + " x " + std::to_string(length) + " operand");
    return data;
}

// (bytes of the rows' operand, of the columns' operand, rows, columns); an operand that is not asked for is None
py::tuple i8_quantize(py::handle x, bool by_rows, bool by_columns)
{
    const Source s = source(tensor(x, "x"), "x");
    if (s.swapped) std::swap(by_rows, by_columns);
    Tensor r = by_rows ? bytes(operand_bytes(s.rows, s.cols), s.t) : Tensor(), c = by_columns ? bytes(operand_bytes(s.cols, s.rows), s.t) : Tensor(), ws;
    const size_t need = by_columns ? amsim_i8_quantize_workspace_bytes(s.rows, s.cols) : 0;
    if (need) ws = bytes((int64_t)need, s.t);
    check(amsim_i8_quantize(s.t.data_ptr(), s.dtype, s.rows, s.cols, s.stride, by_rows ? r.data_ptr() : nullptr, by_columns ? c.data_ptr() : nullptr,
                            need ? ws.data_ptr() : nullptr, need, stream()));
    const py::object a = by_rows ? py::cast(r) : py::none(), b = by_columns ? py::cast(c) : py::none();
    return s.swapped ? py::make_tuple(b, a, s.cols, s.rows) : py::make_tuple(a, b, s.rows, s.cols);
}

Tensor i8_dequantize(py::handle data, int64_t rows, int64_t length, py::handle dtype)
{
    const Tensor &q = operand(tensor(data, "q"), rows, length, "q");
    at::ScalarType t;
    const int code = result_code(dtype, t);
    Tensor out = matrix(rows, length, q, t);
    check(amsim_i8_dequantize(q.data_ptr(), rows, length, code, out.data_ptr(), stream()));
    return out;
}

Tensor i8_matmul(py::handle a_data, int64_t m, py::handle b_data, int64_t n, int64_t k, py::handle bias, int act, py::handle dtype)
{
    const std::optional<Tensor> given_bias = maybe_tensor(bias, "bias");
    if (given_bias) no_derivative(*given_bias, "bias", "int8_matmul", "lineari8");
    const Tensor &a = operand(tensor(a_data, "a"), m, k, "a"), &b = operand(tensor(b_data, "b"), n, k, "b");
    at::ScalarType t;
    const int code = result_code(dtype, t);
    const Bias add = bias_of(given_bias, n, a);
    Tensor out = matrix(m, n, a, t), ws;
    const size_t need = amsim_i8_matmul_workspace_bytes(m, n, k);
    if (need) ws = bytes((int64_t)need, a);
    check(amsim_i8_matmul(a.data_ptr(), b.data_ptr(), m, n, k, add.ptr(), add.dtype, act, out.data_ptr(), code, need ? ws.data_ptr() : nullptr, need, stream()));
    return out;
}

Tensor i8_linear(py::handle given, py::handle data, int64_t n, int64_t k, py::handle bias, int act)
{
    const Tensor &x = tensor(given, "x");
    const std::optional<Tensor> given_bias = maybe_tensor(bias, "bias");
    no_derivative(x, "x", "int8_linear", "lineari8");
    if (given_bias) no_derivative(*given_bias, "bias", "int8_linear", "lineari8");
    if (x.dim() < 1 || x.size(-1) != k) value_error("x's last axis must have the weights' length");
    const Tensor &w = operand(tensor(data, "weights"), n, k, "weights");
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n;
    if (x.numel() == 0) {
        on_device(x, "x"), known(x.scalar_type(), "x");
        bias_of(given_bias, n, x);
        return at::empty(shape, x.options());
    }
    const Source s = row_source(x.dim() == 2 ? x : x.reshape({-1, k}), "x");
    const Bias add = bias_of(given_bias, n, s.t);
    Tensor out = matrix(s.rows, n, s.t, s.t.scalar_type()), ws;
    const size_t need = amsim_i8_linear_workspace_bytes(s.rows, n, k);
    if (need) ws = bytes((int64_t)need, s.t);
    check(amsim_i8_linear(s.t.data_ptr(), s.dtype, s.stride, w.data_ptr(), s.rows, n, k, add.ptr(), add.dtype, act, out.data_ptr(),
                          need ? ws.data_ptr() : nullptr, need, stream()));
    return x.dim() == 2 ? out : out.reshape(shape);
}

// ---- the training step of a layer -------------------------------------------------------------------------------

// What is kept of x and of the kernel, one behind the other in a buffer.
struct Kept {
    int64_t x, kernel;  // bytes of either, 0 where it is not kept
    Kept(int64_t m, int64_t n, int64_t k, bool keep_x, bool keep_kernel)
        : x(keep_x ? (int64_t)amsim_i8_kept_workspace_bytes(k, m) : 0), kernel(keep_kernel ? (int64_t)amsim_i8_kept_workspace_bytes(k, n) : 0)
    {
    }
    int64_t first() const { return (x + 15) / 16 * 16; }
    int64_t all() const { return first() + kernel; }
    uint8_t *of_x(const Tensor &t) const { return x ? (uint8_t *)t.data_ptr() : nullptr; }
    uint8_t *of_kernel(const Tensor &t) const { return kernel ? (uint8_t *)t.data_ptr() + first() : nullptr; }
};

// (the result, what is kept)
std::pair<Tensor, Tensor> dense(const Tensor &given, const Tensor &given_kernel, const std::optional<Tensor> &bias, int act, bool keep_x, bool keep_kernel)
{
    const Source kernel = row_source(given_kernel, "kernel");
    if (given.size(0) == 0) {  // (a batch of nothing, as a router may leave to an expert)
        known(on_device(given, "x").scalar_type(), "x");
        bias_of(bias, kernel.cols, given);
        return {matrix(0, kernel.cols, given, given.scalar_type()), bytes(0, given)};
    }
    const Source x = row_source(given, "x");
    const int64_t m = x.rows, k = x.cols, n = kernel.cols;
    const Bias add = bias_of(bias, n, x.t);
    operand_bytes(m, k), operand_bytes(n, k);
    const Kept keep(m, n, k, keep_x, keep_kernel);
    if (keep_kernel && !keep.kernel) value_error("a layer of " + std::to_string(n) + " units is out of the 8-bit products' range");
    if (keep_x && !keep.x) value_error("a batch of " + std::to_string(m) + " rows is out of the 8-bit products' range");
    const size_t need = amsim_i8_dense_workspace_bytes(m, n, k);
    Tensor out = matrix(m, n, x.t, x.t.scalar_type()), kept, ws = bytes((int64_t)need, x.t);
    if (keep.all()) kept = bytes(keep.all(), x.t);
    check(amsim_i8_dense(x.t.data_ptr(), x.dtype, x.stride, kernel.t.data_ptr(), kernel.dtype, kernel.stride, m, n, k, add.ptr(), add.dtype, act,
                         out.data_ptr(), keep.of_x(kept), keep.of_kernel(kept), ws.data_ptr(), need, stream()));
    return {out, kept};
}

// x is kept as the codes that were multiplied, a byte for each value, and so is the kernel; the backward pass multiplies
// the gradient by them.
struct LinearI8 : torch::autograd::Function<LinearI8> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &kernel, const std::optional<Tensor> &bias, int64_t act, int64_t eager)
    {
        const bool need_x = x.requires_grad(), need_kernel = kernel.requires_grad();
        auto [out, kept] = dense(x, kernel, bias, (int)act, need_kernel, need_x);
        ctx->save_for_backward(act == AMSIM_ACT_RELU ? variable_list{kept, out} : variable_list{kept});
        ctx->saved_data["shape"] = std::vector<int64_t>{x.size(0), x.size(1), kernel.size(1), need_x, need_kernel, (int64_t)kernel.scalar_type(),
                                                        bias && bias->requires_grad() ? (int64_t)bias->scalar_type() : -1, eager};
        return out;
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &given)
    {
        const variable_list saved = ctx->get_saved_variables();
        const std::vector<int64_t> s = ctx->saved_data["shape"].toIntVector();
        const int64_t m = s[0], k = s[1], n = s[2];
        for (int i = 0; i < 3; ++i)
            TORCH_CHECK(!(s[7] >> i & 1) || !ctx->needs_input_grad(i) || !capturing(),
                        "lineari8's backward pass is captured while a graph of the same leaves lives that was made on the default stream, where "
                        "their gradients would be added: release it (its outputs and losses) before the capture");
        const bool want_x = s[3] && ctx->needs_input_grad(0), want_kernel = s[4] && ctx->needs_input_grad(1), want_bias = s[6] >= 0 && ctx->needs_input_grad(2);
        const at::ScalarType kernel_type = (at::ScalarType)s[5], bias_type = want_bias ? (at::ScalarType)s[6] : at::kFloat;
        variable_list grads(5);
        {
            at::AutoGradMode off(false);
            const Tensor &g = given[0];
            const at::TensorOptions like = g.options();
            if (want_x) grads[0] = at::empty({m, k}, like);
            if (want_kernel) grads[1] = m ? at::empty({k, n}, like.dtype(kernel_type)) : at::zeros({k, n}, like.dtype(kernel_type));
            if (want_bias) grads[2] = m ? at::empty({n}, like.dtype(bias_type)) : at::zeros({n}, like.dtype(bias_type));
            if (m) {
                const Source grad = row_source(g, "grad");
                const Kept keep(m, n, k, s[4], s[3]);
                const Tensor &kept = saved[0], none, &out = saved.size() > 1 ? saved[1] : none;
                // (a hook may have brought back something else than was saved)
                auto is = [&](const Tensor &t, at::ScalarType type, int64_t size) {
                    return t.defined() && t.is_cuda() && t.get_device() == grad.t.get_device() && t.scalar_type() == type && t.is_contiguous() && t.numel() == size;
                };
                TORCH_CHECK((!keep.all() || is(kept, at::kByte, keep.all())) && (!out.defined() || is(out, g.scalar_type(), m * n)) && grad.rows == m && grad.cols == n,
                            "what lineari8 kept for its backward pass came back in another form");
                const size_t need = amsim_i8_dense_grad_workspace_bytes(m, n, k);
                Tensor ws = bytes((int64_t)need, grad.t);
                auto ptr = [](const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
                const int status = amsim_i8_dense_grad(grad.t.data_ptr(), grad.dtype, grad.stride, ptr(out), keep.of_x(kept), keep.of_kernel(kept), m, n, k, ptr(grads[0]),
                                                       ptr(grads[1]), code_of(kernel_type), ptr(grads[2]), code_of(bias_type), ws.data_ptr(), need, stream());
                TORCH_CHECK(status == 0, "amsim status ", status, ": ", amsim_last_error());
            }
        }
        no_second_derivative(grads, true, "lineari8");
        return grads;
    }
};

Tensor lineari8(py::handle x_, py::handle kernel_, py::handle bias_, int act)
{
    const Tensor &x = tensor(x_, "x"), &kernel = tensor(kernel_, "kernel");
    const std::optional<Tensor> bias = maybe_tensor(bias_, "bias");
    if (x.dim() < 1 || kernel.dim() != 2 || x.size(-1) != kernel.size(0)) value_error("lineari8 expects x [..., width] and kernel [width, units]");
    if (kernel.numel() == 0) value_error("lineari8 of no elements");
    on_device(x, "x"), on_device(kernel, "kernel");
    if (x._fw_grad(0).defined() || kernel._fw_grad(0).defined() || (bias && bias->_fw_grad(0).defined()))
        type_error("lineari8 has no forward-mode derivative");
    const Tensor flat = x.dim() == 2 ? x : x.reshape({x.numel() ? -1 : 0, x.size(-1)});
    const bool graph = at::GradMode::is_enabled() && (x.requires_grad() || kernel.requires_grad() || (bias && bias->requires_grad()));
    const int64_t eager = graph && capturing() ? adds_on_default_stream(x) | adds_on_default_stream(kernel) << 1 | (bias && adds_on_default_stream(*bias)) << 2 : 0;
    const Tensor out = graph ? LinearI8::apply(flat, kernel, bias, (int64_t)act, eager) : dense(flat, kernel, bias, act, false, false).first;
    if (x.dim() == 2) return out;
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = kernel.size(1);
    return out.reshape(shape);
}

}  // namespace

void amsim_torch::bind_i8(py::module_ &m)
{
    m.def("i8_quantize", &i8_quantize);
    m.def("i8_dequantize", &i8_dequantize);
    m.def("i8_matmul", &i8_matmul);
    m.def("i8_linear", &i8_linear);
    m.def("lineari8", &lineari8);
}
