// The operators over feature rows (linear, layer_norm, dropout) as torch functions with gradients: checks, row views,
// outputs and workspaces here, kernels behind the C ABI.  Part of the compiled extension of torch_ext.cpp, so that
// neither the forward nor the backward pass of a layer runs any Python.
#include <torch/extension.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <dlfcn.h>

#include <climits>
#include <string>

#include "../../include/ngs_rasterizer.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct DecoderApi {
    decltype(&ngs_linear_forward_workspace_bytes) linear_forward_ws = nullptr;
    decltype(&ngs_linear_forward) linear_forward = nullptr;
    decltype(&ngs_linear_backward_workspace_bytes) linear_backward_ws = nullptr;
    decltype(&ngs_linear_slope_bytes) linear_slope_bytes = nullptr;
    decltype(&ngs_linear_backward) linear_backward = nullptr;
    decltype(&ngs_layer_norm_forward) norm_forward = nullptr;
    decltype(&ngs_layer_norm_backward_workspace_bytes) norm_backward_ws = nullptr;
    decltype(&ngs_layer_norm_backward) norm_backward = nullptr;
    decltype(&ngs_dropout) dropout = nullptr;
    decltype(&ngs_last_error) last_error = nullptr;
} api;

void check(int rc) { TORCH_CHECK(rc == 0, api.last_error()); }

int dtype_of(const char* what, const Tensor& t)
{
    switch (t.scalar_type()) {
    case torch::kFloat32: return NGS_FLOAT32;
    case torch::kFloat16: return NGS_FLOAT16;
    case torch::kBFloat16: return NGS_BFLOAT16;
    default: TORCH_CHECK(false, what, ": float32, float16 or bfloat16 expected (got ", t.scalar_type(), ")");
    }
}

// what every operator asks of its first tensor
void check_rows(const char* what, const Tensor& x)
{
    TORCH_CHECK(api.dropout != nullptr, "the rasterizer library has not been bound (call bind(path) first)");
    TORCH_CHECK(x.is_cuda(), what, " runs on the GPU only: x is on ", x.device().str());
    TORCH_CHECK(x.layout() == torch::kStrided, what, ": x must be a dense tensor");
    TORCH_CHECK(x.dim() >= 1, what, ": x must have at least one dimension");
    dtype_of(what, x);
}

// widths that the C entries count in 32 bits (a dropout's rows may be longer: a flat tensor is one)
void check_width(const char* what, const Tensor& x)
{
    TORCH_CHECK(x.size(-1) <= INT_MAX, what, ": rows are too long");
}

void check_like(const char* what, const char* name, const Tensor& t, const Tensor& x, bool float_too = false)
{
    TORCH_CHECK(t.device() == x.device(), what, ": ", name, " must live on ", x.device().str(), " (got ", t.device().str(), ")");
    TORCH_CHECK(t.layout() == torch::kStrided, what, ": ", name, " must be a dense tensor");
    TORCH_CHECK(t.scalar_type() == x.scalar_type() || (float_too && t.scalar_type() == torch::kFloat32), what, ": ", name,
                " must be ", x.scalar_type(), float_too ? " or float32" : "", " (got ", t.scalar_type(), ")");
}

// A tensor as rows of `width` elements that follow each other at a fixed stride; a copy where its strides do not allow
// that (elements of a row not contiguous, leading dimensions that do not collapse) or where its memory holds the
// negated values (torch's lazy negation).
struct Rows {
    Tensor t;
    int64_t rows, width, stride;
};

Rows rows_of(const Tensor& given, int64_t width)
{
    const Tensor x = given.is_neg() ? given.resolve_neg() : given;
    int64_t rows = 1;
    for (int64_t d = 0; d + 1 < x.dim(); d++) rows *= x.size(d);
    Tensor t = x.dim() == 2 ? x : x.reshape({rows, width});
    if (width > 1 && t.stride(1) != 1) t = t.contiguous();
    return {t, rows, width, t.stride(0)};
}

Tensor vec(const Tensor& t) { return t.is_neg() ? t.resolve_neg().contiguous() : t.is_contiguous() ? t : t.contiguous(); }

const void* ptr(const c10::optional<Tensor>& t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }
bool wants_grad(const c10::optional<Tensor>& t) { return t.has_value() && t->defined() && t->requires_grad(); }

hipStream_t stream_of(const Tensor& t)
{
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

Tensor workspace_of(const Tensor& x, size_t bytes)
{
    return bytes ? torch::empty({(int64_t)bytes}, x.options().dtype(torch::kUInt8).requires_grad(false)) : Tensor();
}
char* bytes_ptr(Tensor& t) { return t.defined() ? reinterpret_cast<char*>(t.data_ptr()) : nullptr; }

std::vector<int64_t> with_last(const Tensor& x, int64_t last)
{
    std::vector<int64_t> s = x.sizes().vec();
    s.back() = last;
    return s;
}

void refuse_double_backward(const char* what)
{
    // the engine enables gradients inside a backward pass exactly when a graph of it is asked for
    TORCH_CHECK(!at::GradMode::is_enabled(), what, " has no second derivative (create_graph=True)");
}

// A gradient's accumulator belongs to the stream it was made on.  One that an earlier, eager graph of the same leaf keeps
// alive would make the backward pass wait across streams, which a capture does not survive: refused here, where it can
// still be told.  (The leaf may be what the tensor is a view of: a slice of wider rows, a weight within flat parameters.)
void check_capture(const char* what, const c10::optional<Tensor>& t)
{
    if (!wants_grad(t)) return;
    const Tensor leaf = t->is_leaf() || !t->is_view() ? *t : Tensor(t->_base());
    if (!leaf.is_leaf() || !leaf.requires_grad()) return;
    const auto stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t->device().index());
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream.stream(), &status) != hipSuccess) {
        (void)hipGetLastError();  // not this call's failure to report
        return;
    }
    if (status == hipStreamCaptureStatusNone) return;
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(leaf);
    if (!accumulator) return;
    const auto its = accumulator->stream();
    TORCH_CHECK(!its.has_value() || *its == stream.unwrap(), what,
                ": cannot be captured with gradients while an earlier graph of the same tensor is alive (drop its outputs first)");
}

// ---- linear ----

int activation_of(const std::string& name)
{
    if (name == "none") return NGS_ACT_NONE;
    if (name == "relu") return NGS_ACT_RELU;
    if (name == "gelu") return NGS_ACT_GELU;
    if (name == "silu") return NGS_ACT_SILU;
    if (name == "sigmoid") return NGS_ACT_SIGMOID;
    TORCH_CHECK(false, "linear: unknown activation '", name, "' (none, relu, gelu, silu or sigmoid)");
}

Tensor linear_run(const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias, int act,
                  const c10::optional<Tensor>& residual, Tensor* slope)
{
    const int64_t k = weight.size(1), n = weight.size(0);
    const int dtype = dtype_of("linear", x);
    const c10::DeviceGuard guard(x.device());
    const Rows xr = rows_of(x, k), wr = rows_of(weight, k);
    Rows rr{};
    if (residual.has_value()) rr = rows_of(*residual, n);
    Tensor b;
    if (bias.has_value()) b = vec(*bias);
    Tensor y = torch::empty(with_last(x, n), x.options().requires_grad(false));
    if (slope) *slope = torch::empty({xr.rows, n}, y.options().dtype(torch::kFloat32));
    Tensor ws = workspace_of(x, api.linear_forward_ws(xr.rows, (int)k, (int)n, dtype));
    check(api.linear_forward(xr.rows, (int)k, (int)n, dtype, act, xr.t.data_ptr(), xr.stride, wr.t.data_ptr(), wr.stride,
                             b.defined() ? b.data_ptr() : nullptr, rr.t.defined() ? rr.t.data_ptr() : nullptr, rr.stride,
                             y.data_ptr(), slope ? slope->data_ptr<float>() : nullptr, bytes_ptr(ws), stream_of(x)));
    return y;
}

struct LinearFunction : torch::autograd::Function<LinearFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias,
                          int64_t act, const c10::optional<Tensor>& residual)
    {
        const bool gx = x.requires_grad(), gw = weight.requires_grad(), gb = wants_grad(bias);
        const int64_t k = weight.size(1), n = weight.size(0);
        int64_t rows = 1;
        for (int64_t d = 0; d + 1 < x.dim(); d++) rows *= x.size(d);
        const bool curved = act != NGS_ACT_NONE && (gx || gw || gb);
        const bool keep = curved && api.linear_slope_bytes(rows, (int)k, (int)n, dtype_of("linear", x), (int)act) > 0;
        Tensor slope;
        Tensor y = linear_run(x, weight, bias, (int)act, residual, keep ? &slope : nullptr);
        // each product of the backward pass reads one of the two, the activation's derivative is kept or formed again from
        // all three; what is not needed is not kept alive
        const bool again = curved && !slope.defined();
        ctx->save_for_backward({gw || again ? x : Tensor(), gx || again ? weight : Tensor(),
                                again && bias.has_value() ? *bias : Tensor(), slope});
        ctx->saved_data["act"] = act;
        ctx->saved_data["k"] = weight.size(1);
        ctx->saved_data["n"] = weight.size(0);
        ctx->saved_data["bias"] = bias.has_value();
        ctx->saved_data["residual"] = residual.has_value();
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        refuse_double_backward("linear");
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &slope = saved[3];
        const Tensor& dy = grads[0];
        const int64_t act = ctx->saved_data["act"].toInt(), k = ctx->saved_data["k"].toInt(), n = ctx->saved_data["n"].toInt();
        const bool gx = ctx->needs_input_grad(0), gw = ctx->needs_input_grad(1);
        const bool gb = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
        const int dtype = dtype_of("linear", dy);
        const c10::DeviceGuard guard(dy.device());
        const auto options = dy.options().requires_grad(false);
        Tensor dx, dw, db;
        if (gx || gw || gb) {
            const Rows gr = rows_of(dy, n);
            Rows xr{}, wr{};
            if (x.defined()) xr = rows_of(x, k);
            if (weight.defined()) wr = rows_of(weight, k);
            Tensor b;
            if (bias.defined()) b = vec(bias);
            if (gx) dx = torch::empty(with_last(dy, k), options.memory_format(torch::MemoryFormat::Contiguous));
            if (gw) dw = torch::empty({n, k}, options);
            if (gb) db = torch::empty({n}, options);
            Tensor ws = workspace_of(dy, api.linear_backward_ws(gr.rows, (int)k, (int)n, dtype, (int)act));
            check(api.linear_backward(gr.rows, (int)k, (int)n, dtype, (int)act, x.defined() ? xr.t.data_ptr() : nullptr,
                                      xr.stride, weight.defined() ? wr.t.data_ptr() : nullptr, wr.stride,
                                      b.defined() ? b.data_ptr() : nullptr, slope.defined() ? slope.data_ptr<float>() : nullptr,
                                      gr.t.data_ptr(), gr.stride, gx ? dx.data_ptr() : nullptr, gw ? dw.data_ptr() : nullptr,
                                      gb ? db.data_ptr() : nullptr, bytes_ptr(ws), stream_of(dy)));
        }
        return {dx, dw, db, Tensor(), ctx->saved_data["residual"].toBool() ? dy : Tensor()};
    }
};

Tensor linear(const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias, const std::string& activation,
              const c10::optional<Tensor>& residual)
{
    check_rows("linear", x);
    check_width("linear", x);
    const int act = activation_of(activation);
    check_like("linear", "weight", weight, x);
    TORCH_CHECK(weight.dim() == 2 && weight.size(1) == x.size(-1), "linear: weight must have dimensions (out_features, ",
                x.size(-1), ")");
    TORCH_CHECK(weight.size(0) <= INT_MAX, "linear: too many output features");
    if (bias.has_value()) {
        check_like("linear", "bias", *bias, x);
        TORCH_CHECK(bias->dim() == 1 && bias->size(0) == weight.size(0), "linear: bias must have dimensions (", weight.size(0), ")");
    }
    if (residual.has_value()) {
        check_like("linear", "residual", *residual, x);
        TORCH_CHECK(residual->sizes().vec() == with_last(x, weight.size(0)), "linear: residual must have the output's dimensions");
    }
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || wants_grad(bias) || wants_grad(residual))) {
        for (const auto& t : {c10::optional<Tensor>(x), c10::optional<Tensor>(weight), bias, residual}) check_capture("linear", t);
        return LinearFunction::apply(x, weight, bias, (int64_t)act, residual);
    }
    return linear_run(x, weight, bias, act, residual, nullptr);
}

// ---- layer norm ----

Tensor norm_run(const Tensor& x, const c10::optional<Tensor>& weight, const c10::optional<Tensor>& bias, double eps,
                Tensor* stats)
{
    const int64_t width = x.size(-1);
    const int dtype = dtype_of("layer_norm", x);
    const c10::DeviceGuard guard(x.device());
    const Rows xr = rows_of(x, width);
    Tensor w, b;
    if (weight.has_value()) w = vec(*weight);
    if (bias.has_value()) b = vec(*bias);
    const int wtype = w.defined() ? dtype_of("layer_norm", w) : b.defined() ? dtype_of("layer_norm", b) : dtype;
    Tensor y = torch::empty(x.sizes(), x.options().requires_grad(false).memory_format(torch::MemoryFormat::Contiguous));
    float* st = nullptr;
    if (stats) {
        *stats = torch::empty({2, xr.rows}, y.options().dtype(torch::kFloat32));
        st = stats->data_ptr<float>();
    }
    check(api.norm_forward(xr.rows, (int)width, dtype, wtype, (float)eps, xr.t.data_ptr(), xr.stride,
                           w.defined() ? w.data_ptr() : nullptr, b.defined() ? b.data_ptr() : nullptr, y.data_ptr(), st,
                           st ? st + xr.rows : nullptr, stream_of(x)));
    return y;
}

struct LayerNormFunction : torch::autograd::Function<LayerNormFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const c10::optional<Tensor>& weight,
                          const c10::optional<Tensor>& bias, double eps)
    {
        Tensor stats;
        Tensor y = norm_run(x, weight, bias, eps, &stats);
        ctx->save_for_backward({x, weight.has_value() ? *weight : Tensor(), stats});
        ctx->saved_data["bias"] = bias.has_value();
        ctx->saved_data["wtype"] = (int64_t)(weight.has_value() ? weight->scalar_type()
                                             : bias.has_value() ? bias->scalar_type() : x.scalar_type());
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        refuse_double_backward("layer_norm");
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &stats = saved[2];
        const Tensor& dy = grads[0];
        const int64_t width = x.size(-1);
        // (the engine counts the tensors that are there: without a weight the bias comes second)
        const bool gx = ctx->needs_input_grad(0), gw = weight.defined() && ctx->needs_input_grad(1);
        const bool gb = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(weight.defined() ? 2 : 1);
        const c10::DeviceGuard guard(x.device());
        const Rows xr = rows_of(x, width), gr = rows_of(dy, width);
        const auto options = x.options().requires_grad(false).memory_format(torch::MemoryFormat::Contiguous);
        const auto woptions = options.dtype((c10::ScalarType)ctx->saved_data["wtype"].toInt());
        Tensor w, dx, dw, db;
        if (weight.defined()) w = vec(weight);
        if (gx) dx = torch::empty(x.sizes(), options);
        if (gw) dw = torch::empty({width}, woptions);
        if (gb) db = torch::empty({width}, woptions);
        const int dtype = dtype_of("layer_norm", x);
        const int wtype = woptions.dtype() == torch::kFloat32 ? NGS_FLOAT32 : dtype;
        Tensor ws = workspace_of(x, gw || gb ? api.norm_backward_ws(xr.rows, (int)width, dtype) : 0);
        const float* st = stats.data_ptr<float>();
        check(api.norm_backward(xr.rows, (int)width, dtype, wtype, xr.t.data_ptr(), xr.stride,
                                w.defined() ? w.data_ptr() : nullptr, st, st + xr.rows, gr.t.data_ptr(), gr.stride,
                                gx ? dx.data_ptr() : nullptr, gw ? dw.data_ptr() : nullptr, gb ? db.data_ptr() : nullptr,
                                bytes_ptr(ws), stream_of(x)));
        return {dx, dw, db, Tensor()};
    }
};

Tensor layer_norm(const Tensor& x, const c10::optional<Tensor>& weight, const c10::optional<Tensor>& bias, double eps)
{
    check_rows("layer_norm", x);
    check_width("layer_norm", x);
    for (const auto* t : {&weight, &bias}) {
        if (!t->has_value()) continue;
        const char* name = t == &weight ? "weight" : "bias";
        check_like("layer_norm", name, **t, x, true);
        TORCH_CHECK((*t)->dim() == 1 && (*t)->size(0) == x.size(-1), "layer_norm: ", name, " must have dimensions (", x.size(-1), ")");
    }
    TORCH_CHECK(!weight.has_value() || !bias.has_value() || weight->scalar_type() == bias->scalar_type(),
                "layer_norm: weight and bias must have the same type");
    TORCH_CHECK(eps >= 0, "layer_norm: eps must not be negative");
    if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(weight) || wants_grad(bias))) {
        for (const auto& t : {c10::optional<Tensor>(x), weight, bias}) check_capture("layer_norm", t);
        return LayerNormFunction::apply(x, weight, bias, eps);
    }
    return norm_run(x, weight, bias, eps, nullptr);
}

// ---- dropout ----

Tensor dropout_run(const Tensor& x, double p, int64_t seed, const c10::optional<Tensor>& seed_tensor, int64_t offset,
                   const c10::optional<Tensor>& residual)
{
    const int64_t width = x.size(-1);
    const int dtype = dtype_of("dropout", x);
    const c10::DeviceGuard guard(x.device());
    const Rows xr = rows_of(x, width);
    Rows rr{};
    if (residual.has_value()) rr = rows_of(*residual, width);
    Tensor y = torch::empty(x.sizes(), x.options().requires_grad(false).memory_format(torch::MemoryFormat::Contiguous));
    check(api.dropout(xr.rows, width, dtype, p, (unsigned long long)seed, (const unsigned long long*)ptr(seed_tensor),
                      (unsigned long long)offset, xr.t.data_ptr(), xr.stride, rr.t.defined() ? rr.t.data_ptr() : nullptr,
                      rr.stride, y.data_ptr(), stream_of(x)));
    return y;
}

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, int64_t seed,
                          const c10::optional<Tensor>& seed_tensor, int64_t offset, const c10::optional<Tensor>& residual)
    {
        // (a seed tensor that is changed before the backward pass would name another mask: saved, so that the engine
        // notices and refuses)
        ctx->save_for_backward({seed_tensor.has_value() ? *seed_tensor : Tensor()});
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["residual"] = residual.has_value();
        return dropout_run(x, p, seed, seed_tensor, offset, residual);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        refuse_double_backward("dropout");
        const auto saved = ctx->get_saved_variables();
        Tensor dx;
        if (ctx->needs_input_grad(0))
            dx = dropout_run(grads[0], ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(),
                             saved[0].defined() ? c10::optional<Tensor>(saved[0]) : c10::nullopt,
                             ctx->saved_data["offset"].toInt(), c10::nullopt);
        return {dx, Tensor(), Tensor(), Tensor(), Tensor(), ctx->saved_data["residual"].toBool() ? grads[0] : Tensor()};
    }
};

// a whole number (Python's, or one that says it is, as numpy's do) as 64 bits: what exceeds them is cut off, negative
// ones wrap
int64_t word(const char* name, const pybind11::handle& number)
{
    TORCH_CHECK(PyIndex_Check(number.ptr()) && !THPVariable_Check(number.ptr()), "dropout: ", name, " must be a whole number");
    const auto whole = pybind11::reinterpret_steal<pybind11::object>(PyNumber_Index(number.ptr()));
    if (!whole) throw pybind11::error_already_set();
    return (int64_t)PyLong_AsUnsignedLongLongMask(whole.ptr());
}

Tensor dropout(const Tensor& x, double p, const pybind11::object& seed, const pybind11::object& offset,
               const c10::optional<Tensor>& residual)
{
    check_rows("dropout", x);
    TORCH_CHECK(p >= 0.0 && p <= 1.0, "dropout: p must lie in [0, 1]");
    c10::optional<Tensor> seed_tensor;
    int64_t seed_word = 0;
    if (THPVariable_Check(seed.ptr())) {
        seed_tensor = seed.cast<Tensor>();
        TORCH_CHECK(seed_tensor->scalar_type() == torch::kInt64 && seed_tensor->numel() == 1 && seed_tensor->device() == x.device(),
                    "dropout: a seed tensor must be one int64 on ", x.device().str());
        if (seed_tensor->is_neg()) seed_tensor = seed_tensor->resolve_neg();
    } else {
        seed_word = word("seed", seed);
    }
    const int64_t offset_word = word("offset", offset);
    if (residual.has_value()) {
        check_like("dropout", "residual", *residual, x);
        TORCH_CHECK(residual->sizes() == x.sizes(), "dropout: residual must have the dimensions of x");
    }
    const pybind11::gil_scoped_release release;
    if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(residual))) {
        for (const auto& t : {c10::optional<Tensor>(x), residual}) check_capture("dropout", t);
        return DropoutFunction::apply(x, p, seed_word, seed_tensor, offset_word, residual);
    }
    return dropout_run(x, p, seed_word, seed_tensor, offset_word, residual);
}

template <typename F>
void resolve(F& fn, void* handle, const char* name, const std::string& path)
{
    fn = reinterpret_cast<F>(dlsym(handle, name));
    TORCH_CHECK(fn != nullptr, "symbol ", name, " not found in ", path);
}

}  // namespace

// called by torch_ext.cpp
void ngs_decoder_bind(void* handle, const std::string& path)
{
    resolve(api.linear_forward_ws, handle, "ngs_linear_forward_workspace_bytes", path);
    resolve(api.linear_forward, handle, "ngs_linear_forward", path);
    resolve(api.linear_backward_ws, handle, "ngs_linear_backward_workspace_bytes", path);
    resolve(api.linear_slope_bytes, handle, "ngs_linear_slope_bytes", path);
    resolve(api.linear_backward, handle, "ngs_linear_backward", path);
    resolve(api.norm_forward, handle, "ngs_layer_norm_forward", path);
    resolve(api.norm_backward_ws, handle, "ngs_layer_norm_backward_workspace_bytes", path);
    resolve(api.norm_backward, handle, "ngs_layer_norm_backward", path);
    resolve(api.last_error, handle, "ngs_last_error", path);
    resolve(api.dropout, handle, "ngs_dropout", path);
}

void ngs_decoder_register(pybind11::module_& m)
{
    namespace py = pybind11;
    m.def("linear", &linear, py::arg("x"), py::arg("weight"), py::arg("bias") = py::none(), py::arg("activation") = "none",
          py::arg("residual") = py::none(), py::call_guard<py::gil_scoped_release>());
    m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight") = py::none(), py::arg("bias") = py::none(),
          py::arg("eps") = 1e-5, py::call_guard<py::gil_scoped_release>());
    m.def("dropout", &dropout, py::arg("x"), py::arg("p"), py::arg("seed"), py::arg("offset") = 0,
          py::arg("residual") = py::none());
}
