// Layer normalisation, activations whose input is kept in 8 bits, and the keeping itself on torch tensors: arguments,
// results, workspaces, the stream and the nodes of the autograd graph on top of the C ABI (as amsim_torch.cc for the 4-bit products).
#include "amsim_torch.h"

using namespace amsim_torch;

namespace {

// ---- arguments ----------------------------------------------------------------------------------------------------

void check_rows(const Tensor &x, const char *name)
{
    known(on_device(x, name).scalar_type(), name);
    if (x.dim() < 1 || x.size(-1) == 0) value_error(std::string(name) + " has no last axis to go along");
}
// [..., cols] as a matrix of rows; nothing where there are no rows
std::optional<Source> rows_of(const Tensor &x, const char *name)
{
    check_rows(x, name);
    if (x.numel() == 0) return std::nullopt;
    return row_source(x.dim() == 2 ? x : x.reshape({-1, x.size(-1)}), name);
}
Tensor like_rows(const Source &s) { return matrix(s.rows, s.cols, s.t, s.t.scalar_type()); }
Tensor shaped(const Tensor &flat, const Tensor &x) { return x.dim() == 2 ? flat : flat.reshape(x.sizes()); }

// gamma or beta: one entry per column, of one type
struct Parameters {
    Bias gamma, beta;
    int dtype() const { return gamma.t ? gamma.dtype : beta.dtype; }
};
Parameters parameters(const std::optional<Tensor> &gamma, const std::optional<Tensor> &beta, const Tensor &x)
{
    auto one = [&](const std::optional<Tensor> &t, const char *name) {
        if (!t) return Bias{};
        on_device(*t, name);
        if (t->get_device() != x.get_device()) value_error(std::string(name) + " must be on x's device");
        const int dtype = known(t->scalar_type(), name);
        if (t->dim() != 1 || t->size(0) != x.size(-1)) value_error(std::string(name) + " must have one entry per column of x");
        return Bias{t->_is_zerotensor() ? at::zeros(t->sizes(), t->options()) : t->contiguous().resolve_neg(), dtype};
    };
    Parameters p{one(gamma, "gamma"), one(beta, "beta")};
    if (gamma && beta && p.gamma.dtype != p.beta.dtype) type_error("gamma and beta must be of one type");
    return p;
}
void check_epsilon(double epsilon)
{
    if (!(epsilon >= 0)) value_error("epsilon must not be negative");
}

Tensor kept_buffer(const Source &s)
{
    const size_t n = amsim_kept8_workspace_bytes(s.rows, s.cols);
    if (n == 0) value_error("a " + std::to_string(s.rows) + " x " + std::to_string(s.cols) + " tensor is out of range");
    return bytes((int64_t)n, s.t);
}

// in a backward pass errors are the engine's to report
void check_in_graph(int status) { TORCH_CHECK(status == 0, "amsim status ", status, ": ", amsim_last_error()); }

// eager: of the inputs, by their edges, those whose gradients are added on the default stream
void no_capture(AutogradContext *ctx, int64_t eager, const char *call)
{
    for (int i = 0; i < 3; ++i)
        TORCH_CHECK(!(eager >> i & 1) || !ctx->needs_input_grad(i) || !capturing(), call,
                    "'s backward pass is captured while a graph of the same leaves lives that was made on the default stream, where "
                    "their gradients would be added: release it (its outputs and losses) before the capture");
}

// what a backward pass finds of what was saved (a hook may have brought back something else)
void check_saved(bool good, const char *call) { TORCH_CHECK(good, "what ", call, " kept for its backward pass came back in another form"); }
bool plain(const Tensor &t, const Tensor &like, at::ScalarType type, int64_t n)
{
    return t.defined() && t.is_cuda() && t.get_device() == like.get_device() && t.scalar_type() == type && t.is_contiguous() && t.numel() == n;
}

// ---- layer normalisation ------------------------------------------------------------------------------------------

struct Normed {
    Tensor out, statistics, kept;
};
Normed norm(const Source &s, const Parameters &p, double epsilon, bool statistics, bool keep)
{
    Normed n{like_rows(s), statistics ? matrix(s.rows, 2, s.t, at::kFloat) : Tensor(), keep ? kept_buffer(s) : Tensor()};
    check(amsim_layer_norm(s.t.data_ptr(), s.dtype, s.rows, s.cols, s.stride, p.gamma.ptr(), p.beta.ptr(), p.dtype(), (float)epsilon, n.out.data_ptr(),
                           statistics ? (float *)n.statistics.data_ptr() : nullptr, keep ? n.kept.data_ptr() : nullptr, stream()));
    return n;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const std::optional<Tensor> &gamma, const std::optional<Tensor> &beta, double epsilon,
                          bool keep, int64_t eager)
    {
        const bool need_x = x.requires_grad(), need_gamma = gamma && gamma->requires_grad(), need_beta = beta && beta->requires_grad();
        const Parameters p = parameters(gamma, beta, x);
        const std::optional<Source> s = rows_of(x, "x");
        ctx->saved_data["shape"] = std::vector<int64_t>{need_x, need_gamma, need_beta, gamma.has_value(), keep, eager,
                                                        (int64_t)(gamma ? gamma->scalar_type() : beta ? beta->scalar_type() : at::kFloat), x.size(-1)};
        if (!s) {
            ctx->save_for_backward({});
            return at::empty(x.sizes(), x.options());
        }
        const Normed n = norm(*s, p, epsilon, true, keep);
        variable_list saved{n.statistics, keep ? n.kept : x};
        if (gamma) saved.push_back(*gamma);
        ctx->save_for_backward(saved);
        return n.out;
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &given)
    {
        const variable_list saved = ctx->get_saved_variables();
        const std::vector<int64_t> f = ctx->saved_data["shape"].toIntVector();
        no_capture(ctx, f[5], "layernorm");
        // (an input that is None has no edge: beta's is the second where there is no gamma)
        const bool need_x = f[0] && ctx->needs_input_grad(0), need_gamma = f[1] && ctx->needs_input_grad(1), need_beta = f[2] && ctx->needs_input_grad(1 + f[3]), kept = f[4];
        const at::ScalarType type = (at::ScalarType)f[6];
        variable_list result(6);
        {
            at::AutoGradMode off(false);
            const std::optional<Source> g = rows_of(given[0], "grad");
            auto vector = [&](bool zero) { return zero ? at::zeros({f[7]}, given[0].options().dtype(type)) : at::empty({f[7]}, given[0].options().dtype(type)); };
            if (need_gamma) result[1] = vector(!g);
            if (need_beta) result[2] = vector(!g);
            if (!g) {
                if (need_x) result[0] = at::empty(given[0].sizes(), given[0].options());
            } else {
                if (need_x) result[0] = like_rows(*g);
                const Tensor &of_x = saved[1];
                check_saved(g->cols == f[7] && (!f[3] || (saved[2].defined() && saved[2].scalar_type() == type)) && plain(saved[0], g->t, at::kFloat, 2 * g->rows)
                                && (kept ? plain(of_x, g->t, at::kByte, (int64_t)amsim_kept8_workspace_bytes(g->rows, g->cols))
                                         : of_x.defined() && of_x.is_cuda() && of_x.layout() == at::kStrided && of_x.get_device() == g->t.get_device()
                                               && of_x.scalar_type() == g->t.scalar_type() && of_x.dim() == 2 && of_x.size(0) == g->rows && of_x.size(1) == g->cols),
                            "layernorm");
                const std::optional<Source> x = kept ? std::nullopt : rows_of(of_x, "x");
                const Bias gamma = f[3] ? parameters(saved[2], std::nullopt, given[0]).gamma : Bias{};
                const size_t need = need_gamma || need_beta ? amsim_layer_norm_grad_workspace_bytes(g->rows, g->cols) : 0;
                Tensor ws;
                if (need) ws = bytes((int64_t)need, g->t);
                auto ptr = [](const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
                check_in_graph(amsim_layer_norm_grad(g->t.data_ptr(), g->dtype, g->rows, g->cols, g->stride, x ? x->t.data_ptr() : nullptr, x ? x->stride : 0,
                                                     kept ? saved[1].data_ptr() : nullptr, (const float *)saved[0].data_ptr(), gamma.ptr(), code_of(type),
                                                     ptr(result[0]), ptr(result[1]), ptr(result[2]), ptr(ws), need, stream()));
            }
        }
        no_second_derivative(result, true, "layernorm");
        return result;
    }
};

Tensor layernorm(py::handle x_, py::handle gamma_, py::handle beta_, double epsilon, bool keep)
{
    const Tensor &x = tensor(x_, "x");
    const std::optional<Tensor> gamma = maybe_tensor(gamma_, "gamma"), beta = maybe_tensor(beta_, "beta");
    if (x._fw_grad(0).defined() || (gamma && gamma->_fw_grad(0).defined()) || (beta && beta->_fw_grad(0).defined()))
        type_error("layernorm has no forward-mode derivative");
    check_epsilon(epsilon);
    auto requires = [](const std::optional<Tensor> &t) { return t && t->requires_grad(); };
    if (!at::GradMode::is_enabled() || !(x.requires_grad() || requires(gamma) || requires(beta))) {
        const Parameters p = parameters(gamma, beta, x);
        const std::optional<Source> s = rows_of(x, "x");
        return s ? shaped(norm(*s, p, epsilon, false, false).out, x) : at::empty(x.sizes(), x.options());
    }
    check_rows(x, "x");
    if (gamma) on_device(*gamma, "gamma");
    if (beta) on_device(*beta, "beta");
    int64_t eager = 0;
    if (capturing()) {
        eager = adds_on_default_stream(x);
        if (gamma) eager |= adds_on_default_stream(*gamma) << 1;
        if (beta) eager |= adds_on_default_stream(*beta) << (1 + gamma.has_value());
    }
    if (x.dim() == 2) return LayerNorm::apply(x, gamma, beta, epsilon, keep, eager);
    return LayerNorm::apply(x.reshape({x.numel() ? -1 : 0, x.size(-1)}), gamma, beta, epsilon, keep, eager).reshape(x.sizes());
}

Tensor layer_norm(py::handle x_, py::handle gamma_, py::handle beta_, double epsilon)
{
    const Tensor &x = tensor(x_, "x");
    const std::optional<Tensor> gamma = maybe_tensor(gamma_, "gamma"), beta = maybe_tensor(beta_, "beta");
    no_derivative(x, "x", "layer_norm", "layernorm");
    if (gamma) no_derivative(*gamma, "gamma", "layer_norm", "layernorm");
    if (beta) no_derivative(*beta, "beta", "layer_norm", "layernorm");
    check_epsilon(epsilon);
    const Parameters p = parameters(gamma, beta, x);
    const std::optional<Source> s = rows_of(x, "x");
    return s ? shaped(norm(*s, p, epsilon, false, false).out, x) : at::empty(x.sizes(), x.options());
}

// ---- activations ----------------------------------------------------------------------------------------------------

struct ActivationI8 : torch::autograd::Function<ActivationI8> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, int64_t kind, int64_t eager)
    {
        const std::optional<Source> s = rows_of(x, "x");
        ctx->saved_data["shape"] = std::vector<int64_t>{kind, eager};
        if (!s) {
            ctx->save_for_backward({});
            return at::empty(x.sizes(), x.options());
        }
        Tensor out = like_rows(*s), kept = kept_buffer(*s);
        check(amsim_activation(s->t.data_ptr(), s->dtype, s->rows, s->cols, s->stride, (int)kind, out.data_ptr(), kept.data_ptr(), stream()));
        ctx->save_for_backward({kept});
        return out;
    }

    static variable_list backward(AutogradContext *ctx, const variable_list &given)
    {
        const variable_list saved = ctx->get_saved_variables();
        const std::vector<int64_t> f = ctx->saved_data["shape"].toIntVector();
        no_capture(ctx, f[1], "activationi8");
        variable_list result(3);
        {
            at::AutoGradMode off(false);
            const std::optional<Source> g = rows_of(given[0], "grad");
            result[0] = g ? like_rows(*g) : at::empty(given[0].sizes(), given[0].options());
            if (g) check_saved(plain(saved[0], g->t, at::kByte, (int64_t)amsim_kept8_workspace_bytes(g->rows, g->cols)), "activationi8");
            if (g)
                check_in_graph(amsim_activation_grad(g->t.data_ptr(), g->dtype, g->rows, g->cols, g->stride, saved[0].data_ptr(), (int)f[0],
                                                     result[0].data_ptr(), stream()));
        }
        no_second_derivative(result, true, "activationi8");
        return result;
    }
};

Tensor activationi8(py::handle x_, int kind)
{
    const Tensor &x = tensor(x_, "x");
    if (x._fw_grad(0).defined()) type_error("activationi8 has no forward-mode derivative");
    if (!at::GradMode::is_enabled() || !x.requires_grad()) {
        const std::optional<Source> s = rows_of(x, "x");
        if (!s) return at::empty(x.sizes(), x.options());
        Tensor out = like_rows(*s);
        check(amsim_activation(s->t.data_ptr(), s->dtype, s->rows, s->cols, s->stride, kind, out.data_ptr(), nullptr, stream()));
        return shaped(out, x);
    }
    check_rows(x, "x");
    const int64_t eager = capturing() && adds_on_default_stream(x);
    if (x.dim() == 2) return ActivationI8::apply(x, (int64_t)kind, eager);
    return ActivationI8::apply(x.reshape({x.numel() ? -1 : 0, x.size(-1)}), (int64_t)kind, eager).reshape(x.sizes());
}

// ---- tensors kept in 8 bits -------------------------------------------------------------------------------------------

// (bytes, rows, cols)
py::tuple keep8(py::handle x_)
{
    const Tensor &x = tensor(x_, "x");
    no_derivative(x, "x", "keep8", "a function that keeps its input so");
    const std::optional<Source> s = rows_of(x, "x");
    if (!s) value_error("x is empty: rows of no elements have no scale");
    Tensor kept = kept_buffer(*s);
    check(amsim_activation(s->t.data_ptr(), s->dtype, s->rows, s->cols, s->stride, AMSIM_ACT_NONE, nullptr, kept.data_ptr(), stream()));
    return py::make_tuple(kept, s->rows, s->cols);
}

Tensor kept8_values(py::handle data_, int64_t rows, int64_t cols, py::handle dtype)
{
    const Tensor &data = on_device(tensor(data_, "kept"), "kept");
    const size_t need = amsim_kept8_workspace_bytes(rows, cols);
    if (need == 0 || data.scalar_type() != at::kByte || !data.is_contiguous() || data.numel() != (int64_t)need)
        value_error("kept's data are not those of a " + std::to_string(rows) + " x " + std::to_string(cols) + " tensor");
    at::ScalarType t;
    const int code = result_code(dtype, t);
    Tensor out = matrix(rows, cols, data, t);
    check(amsim_kept8_values(data.data_ptr(), rows, cols, code, out.data_ptr(), stream()));
    return out;
}

}  // namespace

void amsim_torch::bind_rows(py::module_ &m)
{
    m.def("layernorm", &layernorm);
    m.def("layer_norm", &layer_norm);
    m.def("activationi8", &activationi8);
    m.def("keep8", &keep8);
    m.def("kept8_values", &kept8_values);
}
