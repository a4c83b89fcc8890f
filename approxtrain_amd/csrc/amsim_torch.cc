// The 4-bit products and the optimizer's step on torch tensors: checks of arguments, results, workspaces and
// the stream, and the training layer's node of the autograd graph.  Everything that is computed goes through the C ABI.
//
// Small calls take the device fewer microseconds than the interpreter needs to check arguments and to reach the
// library one ctypes call after another: a layer's serving call took 13 us of host time that way and takes 5 to 8 here, the
// training step of a 128 x 784 x 300 layer 125 and 40 to 76 (most of it torch's own engine), functors.adamw_step of 192 tensors 116
// and 12 (the optimizer's step, which gathers the gradients first, 38).
#include "amsim_torch.h"

using namespace amsim_torch;

namespace {

// ---- operands ----------------------------------------------------------------------------------------------------

int64_t operand_bytes(int64_t rows, int64_t length)
{
    const size_t n = amsim_mxfp4_operand_workspace_bytes(rows, length);
    if (n == 0) value_error("a " + std::to_string(rows) + " x " + std::to_string(length) + " tensor is out of the 4-bit products' range");
    return (int64_t)n;
}
// the bytes of an MXTensor
const Tensor &operand(const Tensor &data, int64_t rows, int64_t length, const char *name)
{
    on_device(data, name);
    if (data.scalar_type() != at::kByte || !data.is_contiguous() || data.numel() != operand_bytes(rows, length))
        value_error(std::string(name) + "'s data are not those of a " + std::to_string(rows) + " x " + std::to_string(length) + " operand");
    return data;
}

// ---- conversions and products -----------------------------------------------------------------------------------

// (bytes of the rows' operand, of the columns' operand, rows, columns); an operand that is not asked for is None
py::tuple quantize(py::handle x, bool by_rows, bool by_columns)
{
    const Source s = source(tensor(x, "x"), "x");
    if (s.swapped) std::swap(by_rows, by_columns);
    Tensor r = by_rows ? bytes(operand_bytes(s.rows, s.cols), s.t) : Tensor(), c = by_columns ? bytes(operand_bytes(s.cols, s.rows), s.t) : Tensor();
    check(amsim_mxfp4_quantize(s.t.data_ptr(), s.dtype, s.rows, s.cols, s.stride, by_rows ? r.data_ptr() : nullptr,
                               by_columns ? c.data_ptr() : nullptr, stream()));
    const py::object a = by_rows ? py::cast(r) : py::none(), b = by_columns ? py::cast(c) : py::none();
    return s.swapped ? py::make_tuple(b, a, s.cols, s.rows) : py::make_tuple(a, b, s.rows, s.cols);
}

Tensor dequantize(py::handle data, int64_t rows, int64_t length, py::handle dtype)
{
    const Tensor &q = operand(tensor(data, "q"), rows, length, "q");
    at::ScalarType t;
    const int code = result_code(dtype, t);
    Tensor out = matrix(rows, length, q, t);
    check(amsim_mxfp4_dequantize(q.data_ptr(), rows, length, code, out.data_ptr(), stream()));
    return out;
}

Tensor matmul(py::handle a_data, int64_t m, py::handle b_data, int64_t n, int64_t k, py::handle bias, int act, py::handle dtype)
{
    const std::optional<Tensor> given_bias = maybe_tensor(bias, "bias");
    if (given_bias) no_derivative(*given_bias, "bias", "mxfp4_matmul", "linearmx");
    const Tensor &a = operand(tensor(a_data, "a"), m, k, "a"), &b = operand(tensor(b_data, "b"), n, k, "b");
    at::ScalarType t;
    const int code = result_code(dtype, t);
    const Bias add = bias_of(given_bias, n, a);
    Tensor out = matrix(m, n, a, t), ws;
    const size_t need = amsim_mxfp4_matmul_workspace_bytes(m, n, k);
    if (need) ws = bytes((int64_t)need, a);
    check(amsim_mxfp4_matmul(a.data_ptr(), b.data_ptr(), m, n, k, add.ptr(), add.dtype, act, out.data_ptr(), code, need ? ws.data_ptr() : nullptr, need, stream()));
    return out;
}

Tensor linear(py::handle given, py::handle data, int64_t n, int64_t k, py::handle bias, int act)
{
    const Tensor &x = tensor(given, "x");
    const std::optional<Tensor> given_bias = maybe_tensor(bias, "bias");
    no_derivative(x, "x", "mxfp4_linear", "linearmx");
    if (given_bias) no_derivative(*given_bias, "bias", "mxfp4_linear", "linearmx");
    if (x.dim() < 1 || x.size(-1) != k) value_error("x's last axis must have the weights' length");
    const Tensor &w = operand(tensor(data, "weights"), n, k, "weights");
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n;
    const Tensor flat = x.dim() == 2 ? x : x.reshape({-1, k});
    if (flat.size(0) == 0) {
        on_device(x, "x"), known(x.scalar_type(), "x");
        return at::empty(shape, x.options());
    }
    const Source s = row_source(flat, "x");
    const Bias add = bias_of(given_bias, n, s.t);
    Tensor out = matrix(s.rows, n, s.t, s.t.scalar_type()), ws;
    const size_t need = amsim_mxfp4_linear_workspace_bytes(s.rows, n, k);
    if (need) ws = bytes((int64_t)need, s.t);
    check(amsim_mxfp4_linear(s.t.data_ptr(), s.dtype, s.stride, w.data_ptr(), s.rows, n, k, add.ptr(), add.dtype, act, out.data_ptr(),
                             need ? ws.data_ptr() : nullptr, need, stream()));
    return x.dim() == 2 ? out : out.reshape(shape);
}

// ---- the training step of a layer -------------------------------------------------------------------------------

// (the result, what the backward pass multiplies by)
std::pair<Tensor, Tensor> dense(const Tensor &given, const Tensor &given_kernel, const std::optional<Tensor> &bias, int act, bool keep_x, bool keep_kernel)
{
    const Source kernel = row_source(given_kernel, "kernel");
    if (given.dim() == 2 && given.size(0) == 0) {  // (a batch of nothing, as a router may leave to an expert)
        known(on_device(given, "x").scalar_type(), "x");
        if (kernel.rows != given.size(1)) value_error("the kernel must have as many rows as x has columns");
        bias_of(bias, kernel.cols, given);
        return {matrix(0, kernel.cols, given, given.scalar_type()), bytes(0, given)};
    }
    const Source x = row_source(given, "x");
    const int64_t m = x.rows, k = x.cols, n = kernel.cols;
    if (kernel.rows != k) value_error("the kernel must have as many rows as x has columns");
    const Bias add = bias_of(bias, n, x.t);
    const int64_t x_bytes = operand_bytes(k, m), kernel_bytes = operand_bytes(k, n);
    const size_t need = amsim_mxfp4_dense_workspace_bytes(m, n, k);
    Tensor out = matrix(m, n, x.t, x.t.scalar_type()), kept = bytes((keep_x ? x_bytes : 0) + (keep_kernel ? kernel_bytes : 0), x.t), ws = bytes((int64_t)need, x.t);
    uint8_t *at = (uint8_t *)kept.data_ptr();
    check(amsim_mxfp4_dense(x.t.data_ptr(), x.dtype, x.stride, kernel.t.data_ptr(), kernel.dtype, kernel.stride, m, n, k, add.ptr(), add.dtype, act,
                            out.data_ptr(), keep_x ? at : nullptr, keep_kernel ? at + (keep_x ? x_bytes : 0) : nullptr, ws.data_ptr(), need, stream()));
    return {out, kept};
}

struct Wanted {  // the gradients' types, where they are wanted
    bool x;
    std::optional<at::ScalarType> kernel, bias;
};
// (gradients of x, of the kernel, of the bias); returns the library's status
int dense_grad(const Tensor &given, const Tensor &kept, bool kept_x, bool kept_kernel, int64_t m, int64_t k, int64_t n, const std::optional<Tensor> &out,
               const Wanted &want, Tensor (&grads)[3])
{
    if (m == 0) {
        on_device(given, "grad");
        if (given.dim() != 2 || given.size(0) != 0 || given.size(1) != n) value_error("grad must have the result's shape");
        if (want.x) grads[0] = matrix(0, k, given, given.scalar_type());
        if (want.kernel) grads[1] = at::zeros({k, n}, given.options().dtype(*want.kernel));
        if (want.bias) grads[2] = at::zeros({n}, given.options().dtype(*want.bias));
        return 0;
    }
    const Source grad = row_source(given, "grad");
    if (grad.rows != m || grad.cols != n) value_error("grad must have the result's shape");
    if (out && (out->scalar_type() != grad.t.scalar_type() || out->dim() != 2 || out->size(0) != m || out->size(1) != n || !out->is_contiguous()
                || out->get_device() != grad.t.get_device()))
        value_error("out must be the contiguous result of mxfp4_dense, of grad's type and shape");
    const int64_t x_bytes = kept_x ? operand_bytes(k, m) : 0, kernel_bytes = kept_kernel ? operand_bytes(k, n) : 0;
    if (kept.get_device() != grad.t.get_device() || kept.scalar_type() != at::kByte || !kept.is_contiguous() || kept.numel() != x_bytes + kernel_bytes
        || (want.kernel && !kept_x) || (want.x && !kept_kernel))
        value_error("kept must be what mxfp4_dense returned for these gradients");
    const uint8_t *at = (const uint8_t *)kept.data_ptr();
    if (want.x) grads[0] = matrix(m, k, grad.t, grad.t.scalar_type());
    if (want.kernel) grads[1] = matrix(k, n, grad.t, *want.kernel);
    if (want.bias) grads[2] = at::empty({n}, grad.t.options().dtype(*want.bias));
    const size_t need = amsim_mxfp4_dense_grad_workspace_bytes(m, n, k);
    Tensor ws = bytes((int64_t)need, grad.t);
    auto ptr = [](const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
    return amsim_mxfp4_dense_grad(grad.t.data_ptr(), grad.dtype, grad.stride, out ? out->data_ptr() : nullptr, want.kernel ? at : nullptr,
                                  want.x ? at + x_bytes : nullptr, m, n, k, ptr(grads[0]), ptr(grads[1]), want.kernel ? code_of(*want.kernel) : 0,
                                  ptr(grads[2]), want.bias ? code_of(*want.bias) : 0, ws.data_ptr(), need, stream());
}

py::tuple dense_call(py::handle x, py::handle kernel, py::handle bias, int act, bool keep_x, bool keep_kernel)
{
    const auto got = dense(tensor(x, "x"), tensor(kernel, "kernel"), maybe_tensor(bias, "bias"), act, keep_x, keep_kernel);
    return py::make_tuple(got.first, got.second);
}

py::tuple dense_grad_call(py::handle grad, py::handle kept, int64_t rows, int64_t width, int64_t units, py::handle out, py::handle kernel_dtype,
                          py::handle bias_dtype, bool need_x)
{
    at::ScalarType t;
    Wanted want{need_x, std::nullopt, std::nullopt};
    if (!kernel_dtype.is_none()) result_code(kernel_dtype, t), want.kernel = t;
    if (!bias_dtype.is_none()) result_code(bias_dtype, t), want.bias = t;
    Tensor grads[3];
    check(dense_grad(tensor(grad, "grad"), on_device(tensor(kept, "kept"), "kept"), want.kernel.has_value(), need_x, rows, width, units,
                     maybe_tensor(out, "out"), want, grads));
    auto cast = [](const Tensor &g) { return g.defined() ? py::cast(g) : py::none(); };
    return py::make_tuple(cast(grads[0]), cast(grads[1]), cast(grads[2]));
}

// Each of a layer's three products has its operands quantised along the axis it sums over, so x, the kernel and the
// gradient are quantised both ways, each from one reading; what the backward pass needs is kept in 4 bits.
struct LinearMX : torch::autograd::Function<LinearMX> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &kernel, const std::optional<Tensor> &bias, int64_t act, int64_t eager)
    {
        const bool need_x = x.requires_grad(), need_kernel = kernel.requires_grad();
        auto [out, kept] = dense(x, kernel, bias, (int)act, need_kernel, need_x);
        ctx->save_for_backward(act == AMSIM_ACT_RELU ? variable_list{kept, out} : variable_list{kept});
        ctx->saved_data["shape"] = std::vector<int64_t>{x.size(0), x.size(1), kernel.size(1), need_x, need_kernel, (int64_t)kernel.scalar_type(),
                                                        bias ? (int64_t)bias->scalar_type() : -1, eager};
        return out;
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &given)
    {
        const variable_list saved = ctx->get_saved_variables();
        const std::vector<int64_t> s = ctx->saved_data["shape"].toIntVector();
        Wanted want{s[3] && ctx->needs_input_grad(0), std::nullopt, std::nullopt};
        if (s[4] && ctx->needs_input_grad(1)) want.kernel = (at::ScalarType)s[5];
        if (s[6] >= 0 && ctx->needs_input_grad(2)) want.bias = (at::ScalarType)s[6];
        for (int i = 0; i < 3; ++i)
            TORCH_CHECK(!(s[7] >> i & 1) || !ctx->needs_input_grad(i) || !capturing(),
                        "linearmx's backward pass is captured while a graph of the same leaves lives that was made on the default stream, where "
                        "their gradients would be added: release it (its outputs and losses) before the capture");
        Tensor grads[3];
        {
            at::AutoGradMode off(false);
            const int status = dense_grad(given[0], saved[0], s[4], s[3], s[0], s[1], s[2], saved.size() > 1 ? std::optional<Tensor>(saved[1]) : std::nullopt, want, grads);
            TORCH_CHECK(status == 0, "amsim status ", status, ": ", amsim_last_error());
        }
        variable_list result{grads[0], grads[1], grads[2], Tensor(), Tensor()};
        no_second_derivative(result, given[0].requires_grad(), "linearmx");
        return result;
    }
};

Tensor linearmx(py::handle x_, py::handle kernel_, py::handle bias_, int act)
{
    if (!THPVariable_Check(x_.ptr()) || !THPVariable_Check(kernel_.ptr())) value_error("linearmx expects x [..., width] and kernel [width, units]");
    const Tensor &x = THPVariable_Unpack(x_.ptr()), &kernel = THPVariable_Unpack(kernel_.ptr());
    const std::optional<Tensor> bias = maybe_tensor(bias_, "bias");
    if (x.dim() < 1 || kernel.dim() != 2 || x.size(-1) != kernel.size(0)) value_error("linearmx expects x [..., width] and kernel [width, units]");
    if (kernel.numel() == 0) value_error("linearmx of no elements");
    if (x._fw_grad(0).defined() || kernel._fw_grad(0).defined() || (bias && bias->_fw_grad(0).defined()))
        throw py::type_error("linearmx has no forward-mode derivative");
    const Tensor flat = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
    const bool graph = at::GradMode::is_enabled() && (x.requires_grad() || kernel.requires_grad() || (bias && bias->requires_grad()));
    const int64_t eager = graph && capturing() ? adds_on_default_stream(x) | adds_on_default_stream(kernel) << 1 | (bias && adds_on_default_stream(*bias)) << 2 : 0;
    const Tensor out = graph ? LinearMX::apply(flat, kernel, bias, (int64_t)act, eager) : dense(flat, kernel, bias, act, false, false).first;
    if (x.dim() == 2) return out;
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = kernel.size(1);
    return out.reshape(shape);
}

// ---- AdamW over many tensors --------------------------------------------------------------------------------------

struct TensorList {
    std::vector<int64_t> sizes;
    at::ScalarType dtype;
    int device;

    // pointers of a list of tensors of these sizes, null for None where that may stand
    void pointers(py::list tensors, const char *name, at::ScalarType type, bool none, std::vector<void *> &out) const
    {
        if (tensors.size() != sizes.size()) value_error("as many " + std::string(name) + " as tensors are needed");
        out.resize(sizes.size());
        for (size_t i = 0; i < sizes.size(); ++i) {
            PyObject *o = PyList_GET_ITEM(tensors.ptr(), (Py_ssize_t)i);
            out[i] = nullptr;
            if (none && o == Py_None) continue;
            bool good = THPVariable_Check(o);
            if (good) {
                const Tensor &t = THPVariable_Unpack(o);
                good = t.is_cuda() && t.layout() == at::kStrided && t.scalar_type() == type && t.numel() == sizes[i] && t.get_device() == device
                    && t.is_contiguous() && !t.is_neg() && !t._is_zerotensor();
                if (good) out[i] = t.data_ptr();
            }
            if (!good)
                value_error(std::string(name) + "[" + std::to_string(i) + "] must be a contiguous " + name_of(type) + " tensor of " + std::to_string(sizes[i])
                            + " elements on device " + std::to_string(device));
        }
    }
};

void adamw_step(const TensorList &list, py::list params, py::list grads, int state_bits, py::handle m_, py::handle v_, py::handle m_scale_,
                py::handle v_scale_, int64_t step, double lr, double beta1, double beta2, double eps, double weight_decay, py::handle grad_scale_)
{
    if (grads.size() != params.size()) value_error("as many gradients as parameters are needed");
    if (c10::hip::current_device() != list.device) value_error("the parameters' device is not the current one");
    std::optional<at::ScalarType> grad_type;
    for (py::handle g : grads) {
        if (g.is_none()) continue;
        if (!THPVariable_Check(g.ptr())) value_error("gradients must be tensors or None");
        grad_type = THPVariable_Unpack(g.ptr()).scalar_type();
        break;
    }
    if (!grad_type) return;
    const int grad_code = known(*grad_type, "gradients");
    static thread_local std::vector<void *> p, g;  // (capacity alone outlives a call)
    list.pointers(params, "params", list.dtype, false, p);
    list.pointers(grads, "grads", *grad_type, true, g);
    const Tensor &m = on_device(tensor(m_, "m"), "m"), &v = on_device(tensor(v_, "v"), "v");
    const Tensor &m_scale = on_device(tensor(m_scale_, "m_scale"), "m_scale"), &v_scale = on_device(tensor(v_scale_, "v_scale"), "v_scale");
    int64_t blocks = 0;
    for (int64_t n : list.sizes) blocks += (n + 255) / 256;
    const bool bits8 = state_bits == 8;
    auto holds = [](const Tensor &t, at::ScalarType type, int64_t n) { return t.scalar_type() == type && t.numel() == n && t.is_contiguous(); };
    const at::ScalarType kind = bits8 ? at::kByte : at::kFloat;
    if (!holds(m, kind, blocks * 256) || !holds(v, kind, blocks * 256) || (bits8 && (!holds(m_scale, at::kFloat, blocks) || !holds(v_scale, at::kFloat, blocks))))
        value_error("the state's buffers are not those that AdamWState made");
    const float *scale = nullptr;
    if (!grad_scale_.is_none()) {
        const bool good = THPVariable_Check(grad_scale_.ptr());
        const Tensor s = good ? THPVariable_Unpack(grad_scale_.ptr()) : Tensor();
        if (!good || !s.is_cuda() || s.scalar_type() != at::kFloat || s.numel() != 1 || s.get_device() != list.device || s.is_neg())
            value_error("grad_scale must be one float32 on the parameters' device");
        scale = (const float *)s.data_ptr();
    }
    const amsim_adamw_hyper hyper{step, lr, beta1, beta2, eps, weight_decay};
    check(amsim_adamw_step((int)p.size(), p.data(), (const void *const *)g.data(), list.sizes.data(), code_of(list.dtype), grad_code, state_bits,
                           m.data_ptr(), v.data_ptr(), bits8 ? (float *)m_scale.data_ptr() : nullptr, bits8 ? (float *)v_scale.data_ptr() : nullptr,
                           &hyper, scale, stream()));
    // (written behind autograd's back: a graph that saved a parameter has to notice)
    for (size_t i = 0; i < p.size(); ++i) {
        const Tensor &t = THPVariable_Unpack(PyList_GET_ITEM(params.ptr(), (Py_ssize_t)i));
        if (g[i] && !t.is_inference()) torch::autograd::impl::bump_version(t);
    }
}

// the values that a buffer of 8-bit moments stands for
Tensor state_values(py::handle codes_, py::handle scales_, bool roots)
{
    const Tensor &codes = on_device(tensor(codes_, "codes"), "codes"), &scales = on_device(tensor(scales_, "scales"), "scales");
    if (codes.scalar_type() != at::kByte || scales.scalar_type() != at::kFloat || !codes.is_contiguous() || !scales.is_contiguous()
        || codes.numel() != scales.numel() * 256)
        value_error("moments of 8 bits are bytes in blocks of 256 with a float32 each");
    Tensor out = at::empty({codes.numel()}, codes.options().dtype(at::kFloat));
    if (out.numel()) check(amsim_adamw_state_values(codes.data_ptr(), (const float *)scales.data_ptr(), scales.numel(), roots, (float *)out.data_ptr(), stream()));
    return out;
}

}  // namespace

PYBIND11_MODULE(_native, m)
{
    bind_rows(m);
    bind_i8(m);
    m.def("quantize", &quantize);
    m.def("dequantize", &dequantize);
    m.def("matmul", &matmul);
    m.def("linear", &linear);
    m.def("dense", &dense_call);
    m.def("dense_grad", &dense_grad_call);
    m.def("linearmx", &linearmx);
    m.def("adamw_step", &adamw_step);
    m.def("state_values", &state_values);
    py::class_<TensorList>(m, "TensorList").def(py::init([](std::vector<int64_t> sizes, py::handle dtype, int device) {
        at::ScalarType t;
        result_code(dtype, t);
        return TensorList{std::move(sizes), t, device};
    })).def("check", [](const TensorList &l, py::list tensors, const char *name) {
        std::vector<void *> p;
        l.pointers(tensors, name, l.dtype, false, p);
    });
}
