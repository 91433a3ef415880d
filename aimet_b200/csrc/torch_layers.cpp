// The torch side of the layers: argument checks, memory, streams and autograd around aq_linear_* and aq_layer_norm_*.
// Compiled because a training step of a small layer is bound by the host: the same steps in Python took 143 us for
// forward and backward of a linear layer, 90 of them for the two crossings between autograd's engine and Python.
//
// The C entry points come from the library that the package has loaded (bind()); nothing is linked against it.
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>

#include "../../include/aimet_b200.h"

namespace
{
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library
{
    decltype(&aq_status_string) status_string;
    decltype(&aq_last_cuda_error) last_cuda_error;
    decltype(&aq_align_rows) align_rows;
    decltype(&aq_linear_forward) linear_forward;
    decltype(&aq_linear_grad_z_workspace_bytes) linear_grad_z_workspace_bytes;
    decltype(&aq_linear_grad_z) linear_grad_z;
    decltype(&aq_linear_grad_input) linear_grad_input;
    decltype(&aq_linear_grad_weight) linear_grad_weight;
    decltype(&aq_layer_norm_forward) layer_norm_forward;
    decltype(&aq_layer_norm_backward_workspace_bytes) layer_norm_backward_workspace_bytes;
    decltype(&aq_layer_norm_backward) layer_norm_backward;
} lib = {};

void bind(const py::dict& addresses)
{
    auto get = [&](const char* name, auto& fn) {
        fn = reinterpret_cast<std::decay_t<decltype(fn)>>(addresses[name].cast<uintptr_t>());
    };
    get("aq_status_string", lib.status_string);
    get("aq_last_cuda_error", lib.last_cuda_error);
    get("aq_align_rows", lib.align_rows);
    get("aq_linear_forward", lib.linear_forward);
    get("aq_linear_grad_z_workspace_bytes", lib.linear_grad_z_workspace_bytes);
    get("aq_linear_grad_z", lib.linear_grad_z);
    get("aq_linear_grad_input", lib.linear_grad_input);
    get("aq_linear_grad_weight", lib.linear_grad_weight);
    get("aq_layer_norm_forward", lib.layer_norm_forward);
    get("aq_layer_norm_backward_workspace_bytes", lib.layer_norm_backward_workspace_bytes);
    get("aq_layer_norm_backward", lib.layer_norm_backward);
}

void check(int status, const char* what)
{
    if (status == AQ_OK)
        return;
    TORCH_CHECK(false, "aimet_b200 ", what, " failed: ", lib.status_string(status),
                status == AQ_ERR_CUDA ? std::string(": ") + lib.last_cuda_error() : std::string(), " (status ", status, ")");
}

// ---- arguments ----------------------------------------------------------------------------------------------------
int dtype_of(const Tensor& t)
{
    switch (t.scalar_type())
    {
    case at::kFloat: return AQ_F32;
    case at::kHalf: return AQ_F16;
    case at::kBFloat16: return AQ_BF16;
    default: TORCH_CHECK(false, "aimet_b200: unsupported dtype ", t.scalar_type());
    }
}

void check_input(const Tensor& x)
{
    TORCH_CHECK(x.is_cuda(), "aimet_b200: input must be a CUDA tensor (no CPU path exists), got ", x.device());
    TORCH_CHECK(x.layout() == at::kStrided, "aimet_b200: input must be a dense tensor, got ", x.layout());
    dtype_of(x);
}

void check_operand(const Tensor& t, const Tensor& like, at::IntArrayRef shape, const char* name)
{
    if (!t.defined())
        return;
    TORCH_CHECK(t.sizes() == shape, "aimet_b200: ", name, " must have shape ", shape, ", got ", t.sizes());
    TORCH_CHECK(t.is_cuda(), "aimet_b200: ", name, " must be a CUDA tensor (no CPU path exists), got ", t.device());
    TORCH_CHECK(t.layout() == at::kStrided, "aimet_b200: ", name, " must be a dense tensor, got ", t.layout());
    TORCH_CHECK(t.scalar_type() == like.scalar_type(), "aimet_b200: ", name, " is ", t.scalar_type(), ", the input is ",
                like.scalar_type());
    TORCH_CHECK(t.device() == like.device(), "aimet_b200: tensors on different devices (", like.device(), " vs ", t.device(), ")");
}

// The kernels know nothing of tangents, and a result without one would be taken for a constant.
void check_tangents(std::initializer_list<const Tensor*> tensors)
{
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode())
        return;
    for (const Tensor* t : tensors)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(),
                    "aimet_b200: forward-mode derivatives are not provided for linear and layer_norm");
}

bool wants_grad(std::initializer_list<const Tensor*> tensors)
{
    if (!at::GradMode::is_enabled())
        return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad())
            return true;
    return false;
}

// Memory that holds the tensor's numbers: a lazily negated view's memory holds the others.
Tensor resolved(const Tensor& t)
{
    return t.defined() && t.is_neg() ? t.resolve_neg() : t;
}
// a vector as the kernels read it
Tensor dense(const Tensor& t)
{
    return t.defined() ? resolved(t).contiguous() : t;
}

// `t` as a matrix of rows of `width` elements: a view where rows have unit stride and one pitch, else a copy
Tensor rows_of(const Tensor& t, int64_t width)
{
    Tensor m = resolved(t);
    if (t.dim() != 2 || t.size(1) != width)
        m = m.reshape({m.numel() / width, width});
    if ((width > 1 && m.stride(1) != 1) || (m.size(0) > 1 && m.stride(0) < width))
        m = m.contiguous();
    return m;
}

struct Matrix
{
    void* p    = nullptr;
    int64_t ld = 0;
};
// The stride of a dimension of size 1 can be anything; such a row counts as dense.
Matrix matrix(const Tensor& t)
{
    if (!t.defined())
        return {};
    return {t.data_ptr(), t.size(0) > 1 ? t.stride(0) : (t.size(1) + 7) / 8 * 8};
}

void* ptr(const Tensor& t)
{
    return t.defined() ? t.data_ptr() : nullptr;
}

// Makes x's device current and knows its stream.
struct On
{
    explicit On(const Tensor& x) : guard(x.device()), stream(c10::cuda::getCurrentCUDAStream(x.device().index()).stream())
    {
    }
    c10::cuda::CUDAGuard guard;
    void* stream;
};

// [m, n] whose rows the tensor cores can read
Tensor new_rows(const Tensor& like, int64_t m, int64_t n)
{
    const int64_t pitch = (n + 7) / 8 * 8;
    Tensor t            = at::empty({m, pitch}, like.options());
    return pitch == n ? t : t.narrow(1, 0, n);
}

// `t` itself when the tensor cores can read its rows, else a copy that they can
Tensor aligned_rows(const Tensor& t, const On& on)
{
    if (t.scalar_type() == at::kFloat || t.numel() == 0)
        return t;
    const Matrix m = matrix(t);
    if (reinterpret_cast<uintptr_t>(m.p) % 16 == 0 && m.ld % 8 == 0)
        return t;
    Tensor out     = new_rows(t, t.size(0), t.size(1));
    const Matrix o = matrix(out);
    check(lib.align_rows(m.p, std::max(m.ld, t.size(1)), o.p, o.ld, dtype_of(t), t.size(0), t.size(1), on.stream), "aq_align_rows");
    return out;
}

// Gradients that were formed by the kernels are not differentiable again; asked for with create_graph they say so.
variable_list once(variable_list grads)
{
    if (!at::GradMode::is_enabled())
        return grads;
    variable_list inputs;
    for (const Tensor& g : grads)
        inputs.push_back(g.defined() ? g.detach().requires_grad_(true) : g);
    auto node = std::make_shared<torch::autograd::DelayedError>(
        "aimet_b200: gradients of gradients are not provided for linear and layer_norm", (int64_t) inputs.size());
    variable_list out = node->apply(std::move(inputs));
    for (size_t i = 0; i < grads.size(); ++i)
        if (!grads[i].defined())
            out[i] = Tensor();
    return out;
}

bool needed(AutogradContext* ctx, const char* name)
{
    const int64_t i = ctx->saved_data[name].toInt();
    return i >= 0 && ctx->needs_input_grad((size_t) i);
}

// ---- linear ---------------------------------------------------------------------------------------------------------
struct LinearParts
{
    Tensor y, z, x, w;
};

LinearParts linear_parts(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, int act, bool keep_z)
{
    On on(x);
    const int64_t n = weight.size(0), k = weight.size(1);
    LinearParts r;
    r.x             = rows_of(x, k);
    r.w             = rows_of(weight, k);
    const int64_t m = r.x.size(0);
    if (m > AQ_LINEAR_FEW_ROWS)
    {
        r.x = aligned_rows(r.x, on);
        r.w = aligned_rows(r.w, on);
    }
    const Tensor res = residual.defined() ? rows_of(residual, n) : residual;
    const Tensor b   = dense(bias);
    auto shape       = x.sizes().vec();
    shape.back()     = n;
    r.y              = at::empty(shape, x.options());
    if (keep_z)
        r.z = new_rows(x, m, n);
    if (m)
    {
        const Matrix mx = matrix(r.x), mw = matrix(r.w), mr = matrix(res), mz = matrix(r.z);
        check(lib.linear_forward(mx.p, mx.ld, mw.p, mw.ld, ptr(b), mr.p, mr.ld, r.y.data_ptr(), n, mz.p, mz.ld, dtype_of(x), m, n, k,
                                 act, on.stream),
              "aq_linear_forward");
    }
    return r;
}

// Keeps x, W (their aligned copies where those were made) and, with an activation, z.
struct Linear : torch::autograd::Function<Linear>
{
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias,
                          const std::optional<Tensor>& residual, int64_t act)
    {
        LinearParts r =
            linear_parts(x, weight, bias.value_or(Tensor()), residual.value_or(Tensor()), (int) act, act != AQ_ACT_NONE);
        // the tensors among the arguments are numbered without the missing ones
        ctx->saved_data["bias"]     = bias.has_value() ? 2 : -1;
        ctx->saved_data["residual"] = residual.has_value() ? 2 + (int) bias.has_value() : -1;
        ctx->save_for_backward({weight.requires_grad() ? r.x : Tensor(), x.requires_grad() ? r.w : Tensor(), r.z});
        ctx->saved_data["act"]   = act;
        ctx->saved_data["shape"] = x.sizes();
        ctx->saved_data["n"]     = weight.size(0);
        return r.y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        check_tangents({&grads[0]});
        const bool create_graph = at::GradMode::is_enabled();
        variable_list out(5);
        {
            at::NoGradGuard no_grad;
            const variable_list saved = ctx->get_saved_variables();
            const Tensor &x = saved[0], &w = saved[1], &z = saved[2];
            const auto shape = ctx->saved_data["shape"].toIntVector();
            const int act    = (int) ctx->saved_data["act"].toInt();
            const int64_t n = ctx->saved_data["n"].toInt(), k = shape.back();
            const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = needed(ctx, "bias");
            const Tensor dy = rows_of(grads[0], n);
            const int64_t m = dy.size(0);
            const int dt    = dtype_of(dy);
            On on(dy);
            Tensor dz = dy;
            if (act != AQ_ACT_NONE && (need_x || need_w))
                dz = new_rows(dy, m, n);
            if (need_b || !dz.is_same(dy))
            {
                Tensor ws;
                int64_t bytes = 0;
                if (need_b)
                {
                    out[2] = at::empty({n}, dy.options());
                    bytes  = lib.linear_grad_z_workspace_bytes(dt, m, n);
                    ws     = at::empty({bytes}, dy.options().dtype(at::kByte));
                }
                const Matrix g = matrix(dy), mz = matrix(z), o = dz.is_same(dy) ? Matrix {} : matrix(dz);
                check(lib.linear_grad_z(g.p, g.ld, mz.p, mz.ld, o.p, o.ld, ptr(out[2]), dt, m, n, act, ptr(ws), bytes, on.stream),
                      "aq_linear_grad_z");
            }
            if (need_x || need_w)
                dz = aligned_rows(dz, on);
            const Matrix g = matrix(dz);
            if (need_x)
            {
                out[0] = at::empty(shape, dy.options());
                if (m)
                {
                    const Tensor wa = aligned_rows(w, on);
                    const Matrix mw = matrix(wa);
                    check(lib.linear_grad_input(g.p, g.ld, mw.p, mw.ld, out[0].data_ptr(), k, dt, m, n, k, on.stream),
                          "aq_linear_grad_input");
                }
            }
            if (need_w)
            {
                out[1]          = at::empty({n, k}, dy.options());
                const Tensor xa = aligned_rows(x, on);
                const Matrix mx = matrix(xa);
                check(lib.linear_grad_weight(g.p, g.ld, mx.p, mx.ld, out[1].data_ptr(), k, dt, m, n, k, on.stream),
                      "aq_linear_grad_weight");
            }
        }
        if (create_graph)
            out = once(std::move(out));
        if (needed(ctx, "residual"))
            out[3] = grads[0];
        return out;
    }
};

Tensor linear(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_arg, int64_t act,
              const std::optional<Tensor>& residual_arg)
{
    const Tensor bias = bias_arg.value_or(Tensor()), residual = residual_arg.value_or(Tensor());
    check_tangents({&x, &weight, &bias, &residual});
    check_input(x);
    TORCH_CHECK(weight.dim() == 2 && x.dim() >= 1 && weight.numel() > 0 && x.size(-1) == weight.size(1),
                "aimet_b200: cannot apply a weight of shape ", weight.sizes(), " to an input of shape ", x.sizes());
    const int64_t n = weight.size(0);
    check_operand(weight, x, weight.sizes(), "weight");
    check_operand(bias, x, {n}, "bias");
    if (residual.defined())
    {
        auto shape   = x.sizes().vec();
        shape.back() = n;
        check_operand(residual, x, shape, "residual");
    }
    if (wants_grad({&x, &weight, &bias, &residual}))
        return Linear::apply(x, weight, bias_arg, residual_arg, act);
    return linear_parts(x, weight, bias, residual, (int) act, false).y;
}

// ---- layer norm -------------------------------------------------------------------------------------------------------
struct NormParts
{
    Tensor y, x, w, stats;
};

NormParts norm_parts(const Tensor& x, int64_t dim, const Tensor& weight, const Tensor& bias, double eps, bool keep_stats)
{
    On on(x);
    NormParts r;
    r.x                = rows_of(x, dim);
    r.w                = dense(weight);
    const Tensor b     = dense(bias);
    const int64_t rows = r.x.size(0);
    r.y                = at::empty(x.sizes(), x.options());
    float* mean        = nullptr;
    if (keep_stats)
    {
        r.stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
        mean    = r.stats.data_ptr<float>();
    }
    if (rows)
    {
        const Matrix mx = matrix(r.x);
        check(lib.layer_norm_forward(mx.p, mx.ld, ptr(r.w), ptr(b), r.y.data_ptr(), mean, mean ? mean + rows : nullptr, dtype_of(x),
                                     rows, dim, eps, on.stream),
              "aq_layer_norm_forward");
    }
    return r;
}

// Keeps x and the mean and reciprocal deviation of every row.
struct LayerNorm : torch::autograd::Function<LayerNorm>
{
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight,
                          const std::optional<Tensor>& bias, at::IntArrayRef shape, int64_t dim, double eps)
    {
        NormParts r = norm_parts(x, dim, weight.value_or(Tensor()), bias.value_or(Tensor()), eps, true);
        ctx->saved_data["weight"] = weight.has_value() ? 1 : -1;
        ctx->saved_data["bias"]   = bias.has_value() ? 1 + (int) weight.has_value() : -1;
        ctx->save_for_backward({r.x, r.w, r.stats});
        ctx->saved_data["x"] = x.sizes();
        ctx->saved_data["w"] = shape;
        return r.y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        check_tangents({&grads[0]});
        const bool create_graph = at::GradMode::is_enabled();
        variable_list out(6);
        {
            at::NoGradGuard no_grad;
            const variable_list saved = ctx->get_saved_variables();
            const Tensor &x = saved[0], &w = saved[1];
            const int64_t rows = x.size(0), dim = x.size(1);
            const Tensor dy = rows_of(grads[0], dim);
            On on(dy);
            const int dt = dtype_of(dy);
            if (ctx->needs_input_grad(0))
                out[0] = at::empty(ctx->saved_data["x"].toIntVector(), dy.options());
            if (needed(ctx, "weight"))
                out[1] = at::empty(ctx->saved_data["w"].toIntVector(), dy.options());
            if (needed(ctx, "bias"))
                out[2] = at::empty(ctx->saved_data["w"].toIntVector(), dy.options());
            Tensor ws;
            int64_t bytes = 0;
            if (out[1].defined() || out[2].defined())
            {
                bytes = lib.layer_norm_backward_workspace_bytes(dt, rows, dim);
                ws    = at::empty({bytes}, dy.options().dtype(at::kByte));
            }
            const Matrix mx = matrix(x), mg = matrix(dy);
            const float* mean = saved[2].data_ptr<float>();
            check(lib.layer_norm_backward(mx.p, mx.ld, mg.p, mg.ld, ptr(w), mean, mean + rows, ptr(out[0]), ptr(out[1]), ptr(out[2]),
                                          dt, rows, dim, ptr(ws), bytes, on.stream),
                  "aq_layer_norm_backward");
        }
        return create_graph ? once(std::move(out)) : out;
    }
};

Tensor layer_norm(const Tensor& x, const std::vector<int64_t>& shape, const std::optional<Tensor>& weight_arg,
                  const std::optional<Tensor>& bias_arg, double eps)
{
    const Tensor weight = weight_arg.value_or(Tensor()), bias = bias_arg.value_or(Tensor());
    check_tangents({&x, &weight, &bias});
    check_input(x);
    int64_t dim = 1;
    for (int64_t s : shape)
        dim *= s;
    const int64_t nd = (int64_t) shape.size();
    TORCH_CHECK(nd > 0 && dim > 0 && x.dim() >= nd && x.sizes().slice(x.dim() - nd) == at::IntArrayRef(shape),
                "aimet_b200: cannot normalise an input of shape ", x.sizes(), " over ", at::IntArrayRef(shape));
    TORCH_CHECK(eps >= 0 && std::isfinite(eps), "aimet_b200: eps must be finite and at least 0, got ", eps);
    check_operand(weight, x, shape, "weight");
    check_operand(bias, x, shape, "bias");
    if (wants_grad({&x, &weight, &bias}))
        return LayerNorm::apply(x, weight_arg, bias_arg, at::IntArrayRef(shape), dim, eps);
    return norm_parts(x, dim, weight, bias, eps, false).y;
}
}   // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.def("bind", &bind);
    // without the interpreter's lock, as torch's own functions: a launch waits when the stream's queue is full
    m.def("linear", &linear, py::call_guard<py::gil_scoped_release>());
    m.def("layer_norm", &layer_norm, py::call_guard<py::gil_scoped_release>());
    m.def("rows_of", &rows_of);
}
