// The pybind11 module `train_ops`: the calls of the training operators -- RMS norm, the 8-bit format and its products with
// their gradients, the AdamW step -- from checked arguments to the C entry points on the current stream.  On a single token
// or a small model their kernels take 4 to 10 us, which the same checks, allocations and foreign calls written in Python
// took several times over (one row of 4096: norm with 8-bit output 16.5 us a call from Python, product 11 us, the step of
// ten small tensors 26 us).  `norm.py`, `fp8.py` and `optim.py` call it; it holds nothing from one call to the next.
#include <torch/extension.h>

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <stdexcept>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "gnn_agg.h"
#include "gnn_train.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

constexpr int64_t kBlock = 128;

PyObject *error_class = nullptr;  // the package's GnnAggError

void check_rc(int rc) {
    if (rc == GNNAGG_OK) return;
    // (a backward pass runs on the engine's threads, which do not hold the interpreter)
    TORCH_CHECK(PyGILState_Check(), "libgnnagg error ", rc, ": ", gnnagg_last_error());
    py::object error = py::reinterpret_steal<py::object>(PyObject_CallFunction(error_class, "is", rc, gnnagg_last_error()));
    if (error) PyErr_SetObject(error_class, error.ptr());
    throw py::error_already_set();
}

int64_t padded(int64_t width) { return (width + kBlock - 1) / kBlock * kBlock; }

void check_gpu(const Tensor &t, const char *what) {
    TORCH_CHECK(t.is_cuda(), "Input mismatch: ", what, " must be a GPU (HIP) tensor");
}

void check_gpu(const Tensor &t, const char *what, const Tensor &beside) {
    check_gpu(t, what);
    TORCH_CHECK(t.device() == beside.device(), "Input mismatch: ", what, " is on ", t.device(), ", the other operands on ",
                beside.device());
}

int dtype_code(at::ScalarType type, const char *what) {
    TORCH_CHECK(type == at::kFloat || type == at::kBFloat16, "Input mismatch: ", what,
                " must be float32 or bfloat16, not ", type);
    return type == at::kFloat ? GNNAGG_F32 : GNNAGG_BF16;
}

void refuse_grad(const Tensor &t) {
    TORCH_CHECK(!t.requires_grad(), "this operator has no gradient: use fp8.linear or fp8.norm_linear, or torch.no_grad()");
}

void refuse_grads(std::initializer_list<const OptTensor *> tensors) {
    if (!at::GradMode::is_enabled()) return;
    for (const OptTensor *t : tensors)
        if (t->has_value()) refuse_grad(**t);
}

// The device of a call made current, where it is not, and its stream.
struct Place {
    c10::optional<c10::hip::HIPGuard> guard;
    void *stream;
    explicit Place(const Tensor &t) {
        const auto index = t.device().index();
        if (c10::hip::current_device() != index) guard.emplace(index);
        stream = c10::hip::getCurrentHIPStream(index).stream();
    }
};

bool rows_lie_dense(const Tensor &t) {
    return t.numel() == 0 || ((t.stride(1) == 1 || t.size(1) == 1) && (t.stride(0) >= t.size(1) || t.size(0) == 1));
}

// A tensor as [rows, width] with contiguous rows and a row stride of at least the width: a copy where it has none.
struct Rows {
    Tensor held;
    const void *data;
    int64_t rows, width, stride;
    explicit Rows(const Tensor &t) : held(t), width(t.size(-1)) {
        if (t.dim() == 2 ? rows_lie_dense(t) : width > 0 && t.is_contiguous()) {
            rows = t.dim() == 2 ? t.size(0) : t.numel() / width;
        } else {
            if (t.dim() != 2) held = t.reshape({-1, width});
            if (!rows_lie_dense(held)) held = held.contiguous();
            rows = held.size(0);
        }
        stride = held.dim() == 2 && rows > 1 && width > 0 ? held.stride(0) : std::max<int64_t>(width, 1);
        data = held.const_data_ptr();
    }
};

std::pair<Tensor, Tensor> empty_rows(int64_t rows, int64_t cols, const Tensor &like) {
    const int64_t wide = padded(cols);
    return {at::empty({rows, wide}, like.options().dtype(at::kFloat8_e4m3fn)),
            at::empty({rows, wide / kBlock}, like.options().dtype(at::kFloat8_e8m0fnu))};
}

// What a kernel wrote behind autograd's back counts as changed in place: a backward pass that kept it says so.
void changed(const Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

uint8_t *bytes(const Tensor &t) { return static_cast<uint8_t *>(t.data_ptr()); }

// ------------------------------------------------------------------------------------------------------- RMS norm
struct NormCall {
    Rows x;
    c10::optional<Rows> residual;
    Tensor weight, h;
    int dtype, weight_dtype;
    NormCall(const Tensor &x_, const Tensor &weight_, const OptTensor &residual_) : x(check(x_, weight_, residual_)) {
        dtype = dtype_code(x_.scalar_type(), "x");
        weight = weight_.is_contiguous() ? weight_ : weight_.contiguous();
        weight_dtype = dtype_code(weight.scalar_type(), "the norm's weight");
        if (residual_) {
            residual.emplace(*residual_);
            h = at::empty(x_.sizes(), x_.options());
        }
    }
    static const Tensor &check(const Tensor &x, const Tensor &weight, const OptTensor &residual) {
        check_gpu(x, "x");
        check_gpu(weight, "the norm's weight", x);
        dtype_code(x.scalar_type(), "x");
        TORCH_CHECK(x.dim() >= 1 && weight.dim() == 1 && weight.numel() == x.size(-1),
                    "Input mismatch: the norm's weight must hold one value per column of x");
        TORCH_CHECK(weight.scalar_type() == at::kFloat || weight.scalar_type() == x.scalar_type(),
                    "Input mismatch: the norm's weight must be float32 or of x's type");
        if (residual) {
            check_gpu(*residual, "the residual", x);
            TORCH_CHECK(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(),
                        "Input mismatch: the residual must have x's shape and type");
        }
        return x;
    }
    const void *residual_data() const { return residual ? residual->data : nullptr; }
    int64_t residual_stride() const { return residual ? residual->stride : 0; }
    void *h_data() const { return h.defined() ? h.data_ptr() : nullptr; }
    int64_t h_stride() const { return h.defined() ? x.width : 0; }
    OptTensor stream_rows() const { return h.defined() ? OptTensor(h) : OptTensor(); }
};

// (y, h or None); y: where to write, contiguous rows of x's shape (a column block of a wider array), or None
std::tuple<Tensor, OptTensor> rms_norm(const Tensor &x, const Tensor &weight, double eps, const OptTensor &residual,
                                       bool relu, const OptTensor &y_) {
    const NormCall c(x, weight, residual);
    const Tensor y = y_ ? *y_ : at::empty(x.sizes(), x.options());
    TORCH_CHECK(y.sizes() == x.sizes() && y.scalar_type() == x.scalar_type() && y.device() == x.device() &&
                    (y.is_contiguous() || (y.dim() == 2 && rows_lie_dense(y))),
                "Input mismatch: y must have x's shape and type and contiguous rows");
    const Place place(x);
    check_rc(gnnagg_rms_norm(c.x.data, c.x.stride, c.residual_data(), c.residual_stride(), c.weight.const_data_ptr(),
                             c.weight_dtype, eps, relu, c.h_data(), c.h_stride(), y.data_ptr(),
                             y.dim() == 2 && y.size(0) > 1 && y.size(1) > 0 ? y.stride(0) : std::max<int64_t>(c.x.width, 1),
                             c.x.rows, c.x.width, c.dtype, place.stream));
    if (y_) changed(y);
    return {y, c.stream_rows()};
}

std::tuple<Tensor, Tensor, OptTensor> rms_norm_fp8(const Tensor &x, const Tensor &weight, double eps,
                                                   const OptTensor &residual, bool relu) {
    const NormCall c(x, weight, residual);
    auto [codes, scales] = empty_rows(c.x.rows, c.x.width, x);
    const Place place(x);
    check_rc(gnnagg_rms_norm_fp8(c.x.data, c.x.stride, c.residual_data(), c.residual_stride(), c.weight.const_data_ptr(),
                                 c.weight_dtype, eps, relu, c.h_data(), c.h_stride(), bytes(codes), bytes(scales), c.x.rows,
                                 c.x.width, c.dtype, place.stream));
    return {codes, scales, c.stream_rows()};
}

// -------------------------------------------------------------------------------------------------- 8-bit products
std::tuple<Tensor, Tensor> quantize_rows(const Tensor &x) {
    check_gpu(x, "x");
    const int code = dtype_code(x.scalar_type(), "x");
    TORCH_CHECK(x.dim() == 2 && x.size(1) > 0, "Input mismatch: x must be [rows, width] with a width above zero");
    const Rows rows(x);
    auto [codes, scales] = empty_rows(rows.rows, rows.width, x);
    const Place place(x);
    check_rc(gnnagg_fp8_quantize_rows(rows.data, rows.stride, bytes(codes), bytes(scales), rows.rows, rows.width, code,
                                      place.stream));
    return {codes, scales};
}

typedef std::pair<uintptr_t, uintptr_t> Span;  // of addresses, the end behind it

Span span_of(const Tensor &t) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(t.const_data_ptr());
    return {at, at + t.nbytes()};
}

// Whether a contiguous operand shares bytes with rows [rows, cols] of `out`; columns of a wider array beside them do not
// count.
bool shares_memory(const Tensor &out, const Tensor &operand) {
    if (out.numel() == 0 || operand.numel() == 0) return false;
    const Span s = span_of(operand);
    const uintptr_t at = reinterpret_cast<uintptr_t>(out.const_data_ptr()), size = out.element_size();
    const uintptr_t width = size * out.size(1), pitch = out.size(0) > 1 ? size * out.stride(0) : width;
    if (s.second <= at || s.first >= at + (out.size(0) - 1) * pitch + width) return false;
    if (s.first < at) return true;
    const uintptr_t in_row = (s.first - at) % pitch;       // the row that s begins in, or behind
    return in_row < width || s.first - in_row + pitch < s.second;
}

void check_rows(const Tensor &codes, const Tensor &scales, int64_t cols) {
    check_gpu(codes, "x");
    check_gpu(scales, "x' scales", codes);
    TORCH_CHECK(codes.scalar_type() == at::kFloat8_e4m3fn && codes.dim() == 2 && cols >= 1 &&
                    codes.size(1) == padded(cols) && codes.is_contiguous() &&
                    reinterpret_cast<uintptr_t>(codes.const_data_ptr()) % 16 == 0,
                "Input mismatch: x must hold contiguous, 16-byte aligned float8_e4m3fn codes [rows, cols rounded up to 128]");
    TORCH_CHECK(scales.scalar_type() == at::kFloat8_e8m0fnu && scales.dim() == 2 && scales.size(0) == codes.size(0) &&
                    scales.size(1) == codes.size(1) / kBlock && scales.is_contiguous(),
                "Input mismatch: x must hold contiguous float8_e8m0fnu scales [rows, blocks of 128]");
}

// x @ w (+ bias) or, with input_gradient, x @ w^T; w_codes by output or by input accordingly
Tensor product(const Tensor &x, const Tensor &x_scales, int64_t cols, const OptTensor &w_codes, const Tensor &w_scales,
               int64_t k, int64_t n, const OptTensor &bias_, at::ScalarType out_dtype, const OptTensor &out_,
               bool input_gradient) {
    check_rows(x, x_scales, cols);
    const int64_t rows = x.size(0), inner = input_gradient ? n : k, wide = input_gradient ? k : n;
    TORCH_CHECK(w_codes, "Input mismatch: the weight was quantised without the codes this product reads");
    check_gpu(*w_codes, "the weight", x);
    check_gpu(w_scales, "the weight's scales", x);
    TORCH_CHECK(cols == inner, "Input mismatch: x has ", cols, " columns, the weight's inner width is ", inner);
    TORCH_CHECK(w_codes->scalar_type() == at::kFloat8_e4m3fn && w_codes->dim() == 2 && w_codes->size(0) == wide &&
                    w_codes->size(1) == padded(inner) && w_codes->is_contiguous() &&
                    reinterpret_cast<uintptr_t>(w_codes->const_data_ptr()) % 16 == 0,
                "Input mismatch: the weight must hold contiguous, 16-byte aligned float8_e4m3fn codes [outputs, inner width "
                "rounded up to 128]");
    TORCH_CHECK(w_scales.scalar_type() == at::kFloat8_e8m0fnu && w_scales.dim() == 2 &&
                    w_scales.size(0) == padded(k) / kBlock && w_scales.size(1) == padded(n) / kBlock,
                "Input mismatch: the weight must hold float8_e8m0fnu scales [k blocks, n blocks]");
    const int code = dtype_code(out_ ? out_->scalar_type() : out_dtype, "out");
    Tensor bias;
    if (bias_) {
        check_gpu(*bias_, "the bias", x);
        TORCH_CHECK(bias_->numel() == wide, "Input mismatch: the bias holds ", bias_->numel(), " values for ", wide, " outputs");
        bias = bias_->detach().reshape({-1}).to(at::kFloat).contiguous();
    }
    if (out_) {
        check_gpu(*out_, "out", x);
        TORCH_CHECK(out_->dim() == 2 && out_->size(0) == rows && out_->size(1) == wide && rows_lie_dense(*out_),
                    "Input mismatch: out must be [rows, outputs] with contiguous rows");
        for (const Tensor *t : std::initializer_list<const Tensor *>{&x, &x_scales, &*w_codes, &w_scales, &bias})
            TORCH_CHECK(!t->defined() || !shares_memory(*out_, *t), "Input mismatch: out shares memory with an operand");
    }
    const Tensor out = out_ ? *out_ : at::empty({rows, wide}, x.options().dtype(out_dtype));
    const Place place(x);
    const int64_t stride0 = w_scales.stride(0), stride1 = w_scales.stride(1);
    check_rc(gnnagg_fp8_product(bytes(x), bytes(x_scales), bytes(*w_codes), bytes(w_scales),
                                input_gradient ? stride1 : stride0, input_gradient ? stride0 : stride1,
                                bias.defined() ? bias.const_data_ptr<float>() : nullptr, out.data_ptr(),
                                rows > 1 && wide > 0 ? out.stride(0) : std::max<int64_t>(wide, 1), code, rows, inner, wide,
                                place.stream));
    if (out_) changed(out);
    return out;
}

Tensor public_product(const Tensor &x, const Tensor &x_scales, int64_t cols, const OptTensor &w_codes,
                      const Tensor &w_scales, int64_t k, int64_t n, const OptTensor &bias, at::ScalarType out_dtype,
                      const OptTensor &out, bool input_gradient) {
    refuse_grads({&bias, &out});
    return product(x, x_scales, cols, w_codes, w_scales, k, n, bias, out_dtype, out, input_gradient);
}

std::tuple<Tensor, Tensor> public_quantize_rows(const Tensor &x) {
    if (at::GradMode::is_enabled()) refuse_grad(x);
    return quantize_rows(x);
}

std::tuple<Tensor, Tensor, OptTensor> public_rms_norm_fp8(const Tensor &x, const Tensor &weight, double eps,
                                                          const OptTensor &residual, bool relu) {
    if (at::GradMode::is_enabled()) {
        refuse_grad(x);
        refuse_grad(weight);
        refuse_grads({&residual});
    }
    return rms_norm_fp8(x, weight, eps, residual, relu);
}

// (codes by output, codes by input, scales), either codes where asked for; a weight stored by output is read where it lies
std::tuple<OptTensor, OptTensor, Tensor> quantize_weight(const Tensor &w_, bool by_output, bool by_input) {
    check_gpu(w_, "the weight");
    const int code = dtype_code(w_.scalar_type(), "the weight");
    TORCH_CHECK(w_.dim() == 2 && w_.numel() > 0, "Input mismatch: the weight must be [k, n], neither zero");
    const int64_t k = w_.size(0), n = w_.size(1);
    if (w_.stride(1) != 1 && w_.stride(0) == 1 && w_.stride(1) >= k) {  // its transpose with the roles exchanged
        auto [codes, codes_by_input, scales] = quantize_weight(w_.t(), by_input, by_output);
        return {codes_by_input, codes, scales.t()};
    }
    const Rows w(w_);
    OptTensor codes, codes_by_input;
    const auto type = w_.options().dtype(at::kFloat8_e4m3fn);
    if (by_output) codes = at::empty({n, padded(k)}, type);
    if (by_input) codes_by_input = at::empty({k, padded(n)}, type);
    const Tensor scales = at::empty({padded(k) / kBlock, padded(n) / kBlock}, type.dtype(at::kFloat8_e8m0fnu));
    const Place place(w_);
    check_rc(gnnagg_fp8_quantize_weight(w.data, w.stride, codes ? bytes(*codes) : nullptr,
                                        codes_by_input ? bytes(*codes_by_input) : nullptr, bytes(scales), k, n, code,
                                        place.stream));
    return {codes, codes_by_input, scales};
}

std::tuple<OptTensor, OptTensor, Tensor> public_quantize_weight(const Tensor &w, bool by_input) {
    if (at::GradMode::is_enabled()) refuse_grad(w);
    return quantize_weight(w, true, by_input);
}

// (x^T bf16(g), g's column sums or None)
std::tuple<Tensor, OptTensor> weight_gradient(const Tensor &x, const Tensor &x_scales, int64_t k, const Tensor &g_,
                                              bool with_bias) {
    check_rows(x, x_scales, k);
    check_gpu(g_, "g", x);
    const int code = dtype_code(g_.scalar_type(), "g");
    TORCH_CHECK(g_.dim() == 2 && g_.size(0) == x.size(0) && g_.size(1) > 0, "Input mismatch: g must be [rows of x, outputs]");
    const Rows g(g_);
    const int64_t rows = g.rows, n = g.width;
    const auto type = x.options().dtype(at::kFloat);
    const int64_t nbytes = gnnagg_fp8_weight_gradient_workspace_bytes(rows, k, n);
    const Tensor grad_w = at::empty({k, n}, type);
    OptTensor grad_b;
    if (with_bias) grad_b = at::empty({n}, type);
    Tensor workspace;
    if (nbytes) workspace = at::empty({nbytes}, type.dtype(at::kByte));
    const Place place(x);
    check_rc(gnnagg_fp8_weight_gradient(bytes(x), bytes(x_scales), g.data, g.stride, code, grad_w.data_ptr<float>(),
                                        grad_b ? grad_b->data_ptr<float>() : nullptr, nbytes ? workspace.data_ptr() : nullptr,
                                        nbytes, rows, k, n, place.stream));
    return {grad_w, grad_b};
}

std::tuple<Tensor, OptTensor> public_weight_gradient(const Tensor &x, const Tensor &x_scales, int64_t k, const Tensor &g,
                                                     bool with_bias) {
    if (at::GradMode::is_enabled()) refuse_grad(g);
    return weight_gradient(x, x_scales, k, g, with_bias);
}

// (gradient of x and of the residual, gradient of the weight in its type)
std::tuple<Tensor, Tensor> rms_norm_backward(const Tensor &grad_y_, const OptTensor &grad_h_, const Tensor &h_,
                                             const Tensor &weight_, double eps, bool relu) {
    const Rows grad_y(grad_y_), h(h_);
    c10::optional<Rows> grad_h;
    if (grad_h_) grad_h.emplace(*grad_h_);
    const Tensor weight = weight_.is_contiguous() ? weight_ : weight_.contiguous();
    const int64_t nbytes = gnnagg_rms_norm_backward_workspace_bytes(h.rows, h.width);
    const Tensor grad_x = at::empty(h_.sizes(), h_.options()), grad_w = at::empty({h.width}, h_.options().dtype(at::kFloat));
    const Tensor workspace = at::empty({nbytes}, h_.options().dtype(at::kByte));
    const Place place(h_);
    check_rc(gnnagg_rms_norm_backward(grad_y.data, grad_y.stride, grad_h ? grad_h->data : nullptr,
                                      grad_h ? grad_h->stride : 0, h.data, h.stride, weight.const_data_ptr(),
                                      dtype_code(weight.scalar_type(), "the norm's weight"), eps, relu, grad_x.data_ptr(),
                                      h.width, grad_w.data_ptr<float>(), workspace.data_ptr(), nbytes, h.rows, h.width,
                                      dtype_code(h_.scalar_type(), "x"), place.stream));
    return {grad_x, grad_w.to(weight_.scalar_type())};
}

// ---------------------------------------------------------------------------------------------- differentiable forms
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A gradient's own gradient is refused when it is asked for.
variable_list once_differentiable(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    auto refuse = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that is differentiable once", (int64_t)grads.size());
    for (Tensor &t : grads)
        if (t.defined()) t = t.detach().set_requires_grad(true);  // (so that there is something to refuse)
    return (*refuse)(std::move(grads));
}

OptTensor given(const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }

struct ProductGradients {
    Tensor x, w, b;
};

// gradients of rows @ weight + bias, each where it is wanted
ProductGradients product_gradients(const Tensor &codes, const Tensor &scales, const Tensor &by_input, const Tensor &w_scales,
                                   int64_t k, const Tensor &g, bool want_x, bool want_w, bool want_b, at::ScalarType x_type,
                                   at::ScalarType w_type, at::ScalarType b_type) {
    ProductGradients grads;
    Tensor g_codes, g_scales;
    if (want_x) std::tie(g_codes, g_scales) = quantize_rows(g);  // (both passes over g beside each other)
    if (want_w || want_b) {  // (the bias's sums come with the weight gradient's pass, beside a frozen weight too)
        auto [w, b] = weight_gradient(codes, scales, k, g, want_b);
        if (want_w) grads.w = w.to(w_type);
        if (want_b) grads.b = b->to(b_type);
    }
    if (want_x)
        grads.x = product(g_codes, g_scales, g.size(1), by_input, w_scales, k, g.size(1), OptTensor(), x_type, OptTensor(), true);
    return grads;
}

void check_linear(const Tensor &x, const Tensor &w, const OptTensor &bias) {
    check_gpu(x, "x");
    check_gpu(w, "the weight", x);
    dtype_code(x.scalar_type(), "x");
    dtype_code(w.scalar_type(), "the weight");
    TORCH_CHECK(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(0) && w.numel() > 0, "Input mismatch: x ", x.sizes(),
                " against a weight ", w.sizes());
    if (bias) {
        check_gpu(*bias, "the bias", x);
        dtype_code(bias->scalar_type(), "the bias");
        TORCH_CHECK(bias->dim() == 1 && bias->numel() == w.size(1), "Input mismatch: the bias must hold one value per output");
    }
}

std::vector<int64_t> with_last(at::IntArrayRef sizes, int64_t last) {
    std::vector<int64_t> shape(sizes.begin(), sizes.end());
    shape.back() = last;
    return shape;
}

Tensor flat(const Tensor &t) { return t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}); }

bool wanted(const OptTensor &t) { return at::GradMode::is_enabled() && t && t->requires_grad(); }

struct LinearFunction : torch::autograd::Function<LinearFunction> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const OptTensor &bias, bool for_x) {
        auto [codes, scales] = quantize_rows(flat(x));
        auto [w_codes, by_input, w_scales] = quantize_weight(w, true, for_x);
        const Tensor out = product(codes, scales, w.size(0), w_codes, w_scales, w.size(0), w.size(1), bias, x.scalar_type(),
                                   OptTensor(), false);
        ctx->save_for_backward({codes, scales, by_input ? *by_input : Tensor(), w_scales});
        ctx->saved_data["shape"] = x.sizes().vec();
        ctx->saved_data["types"] = std::vector<int64_t>{(int64_t)x.scalar_type(), (int64_t)w.scalar_type(),
                                                        bias ? (int64_t)bias->scalar_type() : -1};
        return x.dim() == 2 ? out : out.view(with_last(x.sizes(), w.size(1)));
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        const auto saved = ctx->get_saved_variables();
        const auto shape = ctx->saved_data["shape"].toIntVector(), types = ctx->saved_data["types"].toIntVector();
        const bool has_bias = types[2] >= 0;
        const auto grads = product_gradients(saved[0], saved[1], saved[2], saved[3], shape.back(), flat(g[0]),
                                             ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                             has_bias && ctx->needs_input_grad(2), (at::ScalarType)types[0],
                                             (at::ScalarType)types[1], (at::ScalarType)types[2]);
        return once_differentiable({grads.x.defined() && shape.size() != 2 ? grads.x.view(shape) : grads.x, grads.w, grads.b,
                                    Tensor()});
    }
};

Tensor linear(const Tensor &x, const Tensor &w, const OptTensor &bias) {
    check_linear(x, w, bias);
    return LinearFunction::apply(x, w, bias, wanted(x));
}

struct RmsNormFunction : torch::autograd::Function<RmsNormFunction> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const OptTensor &residual, const Tensor &weight,
                                 double eps, bool relu) {
        auto [y, h] = rms_norm(x, weight, eps, residual, relu, OptTensor());
        ctx->save_for_backward({h ? *h : x, weight});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["relu"] = relu;
        ctx->set_materialize_grads(false);
        return h ? variable_list{y, *h} : variable_list{y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        const auto saved = ctx->get_saved_variables();
        const bool has_residual = g.size() == 2;
        Tensor grad_x = has_residual ? g[1] : Tensor(), grad_w;  // (only the residual stream was used)
        if (g[0].defined())
            std::tie(grad_x, grad_w) = rms_norm_backward(g[0], given(grad_x), saved[0], saved[1],
                                                         ctx->saved_data["eps"].toDouble(), ctx->saved_data["relu"].toBool());
        const bool for_x = ctx->needs_input_grad(0), for_residual = has_residual && ctx->needs_input_grad(1);
        const bool for_weight = ctx->needs_input_grad(has_residual ? 2 : 1);
        return once_differentiable({for_x ? grad_x : Tensor(), for_residual ? grad_x : Tensor(),
                                    for_weight ? grad_w : Tensor(), Tensor(), Tensor()});
    }
};

std::tuple<Tensor, Tensor> differentiable_rms_norm(const Tensor &x, const Tensor &weight, double eps, const OptTensor &residual,
                                                   bool relu) {
    NormCall::check(x, weight, residual);
    const auto out = RmsNormFunction::apply(x, residual, weight, eps, relu);
    return {out[0], residual ? out[1] : x};
}

struct NormLinearFunction : torch::autograd::Function<NormLinearFunction> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const OptTensor &residual, const Tensor &norm_weight,
                                 const Tensor &w, const OptTensor &bias, double eps, bool relu, bool for_rows) {
        auto [codes, scales, h] = rms_norm_fp8(x, norm_weight, eps, residual, relu);
        auto [w_codes, by_input, w_scales] = quantize_weight(w, true, for_rows);
        Tensor out = product(codes, scales, w.size(0), w_codes, w_scales, w.size(0), w.size(1), bias, x.scalar_type(),
                             OptTensor(), false);
        ctx->save_for_backward({h ? *h : x, norm_weight, codes, scales, by_input ? *by_input : Tensor(), w_scales});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["relu"] = relu;
        ctx->saved_data["types"] = std::vector<int64_t>{(int64_t)x.scalar_type(), (int64_t)w.scalar_type(),
                                                        bias ? (int64_t)bias->scalar_type() : -1};
        ctx->set_materialize_grads(false);
        if (x.dim() != 2) out = out.view(with_last(x.sizes(), w.size(1)));
        return h ? variable_list{out, *h} : variable_list{out};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        const auto saved = ctx->get_saved_variables();
        const auto types = ctx->saved_data["types"].toIntVector();
        const bool has_residual = g.size() == 2, has_bias = types[2] >= 0;
        const int at = has_residual ? 1 : 0;
        const bool for_x = ctx->needs_input_grad(0), for_residual = has_residual && ctx->needs_input_grad(1);
        const bool for_norm = ctx->needs_input_grad(1 + at), for_w = ctx->needs_input_grad(2 + at);
        const bool for_bias = has_bias && ctx->needs_input_grad(3 + at);
        ProductGradients grads;
        Tensor grad_x = has_residual ? g[1] : Tensor(), grad_norm;
        if (g[0].defined()) {
            grads = product_gradients(saved[2], saved[3], saved[4], saved[5], saved[0].size(-1), flat(g[0]),
                                      for_x || for_residual || for_norm, for_w, for_bias, (at::ScalarType)types[0],
                                      (at::ScalarType)types[1], (at::ScalarType)types[2]);
            if (grads.x.defined())
                std::tie(grad_x, grad_norm) = rms_norm_backward(grads.x, given(grad_x), saved[0], saved[1],
                                                                ctx->saved_data["eps"].toDouble(),
                                                                ctx->saved_data["relu"].toBool());
        }
        return once_differentiable({for_x ? grad_x : Tensor(), for_residual ? grad_x : Tensor(),
                                    for_norm ? grad_norm : Tensor(), grads.w, grads.b, Tensor(), Tensor(), Tensor()});
    }
};

std::tuple<Tensor, Tensor> norm_linear(const Tensor &x, const Tensor &norm_weight, double eps, const Tensor &w,
                                       const OptTensor &bias, const OptTensor &residual, bool relu) {
    NormCall::check(x, norm_weight, residual);
    check_linear(x, w, bias);
    const auto out = NormLinearFunction::apply(x, residual, norm_weight, w, bias, eps, relu,
                                               wanted(x) || wanted(residual) || wanted(norm_weight));
    return {out[0], residual ? out[1] : x};
}

// ----------------------------------------------------------------------------------------------------------- AdamW
typedef std::vector<Tensor> Tensors;

at::ScalarType same(const Tensors &tensors, std::initializer_list<at::ScalarType> types, const Tensors &params,
                    const char *what) {
    TORCH_CHECK(tensors.size() == params.size(), "Input mismatch: ", tensors.size(), " ", what, " for ", params.size(),
                " parameters");
    const auto type = tensors[0].scalar_type();
    TORCH_CHECK(std::find(types.begin(), types.end(), type) != types.end(), "Input mismatch: ", what, " cannot be ", type);
    for (const Tensor &t : tensors) {
        TORCH_CHECK(t.scalar_type() == type, "Input mismatch: ", what, " must all have one type");
        TORCH_CHECK(t.device() == params[0].device(), "Input mismatch: ", what,
                    " must be on the parameters' GPU (HIP) device");
        TORCH_CHECK(t.is_contiguous(), "Input mismatch: ", what, " must be contiguous");
    }
    return type;
}

void same_sizes(const Tensors &tensors, const Tensors &params, const char *what, int64_t block = 1) {
    for (size_t i = 0; i < params.size(); ++i)
        TORCH_CHECK(tensors[i].numel() == (params[i].numel() + block - 1) / block, "Input mismatch: ", what,
                    " number ", i, block == 1 ? " has another size than its parameter"
                                              : " does not hold one value for each 128 elements of its state");
}

// No byte may be written twice, and none that is written may be read as something else: blocks would race for it.
void refuse_overlaps(std::initializer_list<const Tensors *> written, std::initializer_list<const Tensors *> read) {
    std::vector<Span> spans;
    for (const Tensors *tensors : written)
        for (const Tensor &t : *tensors)
            if (t.numel() > 0) spans.push_back(span_of(t));
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
        TORCH_CHECK(spans[i].first >= spans[i - 1].second,
                    "Input mismatch: the same memory twice among parameters, states, masters and steps");
    for (const Tensors *tensors : read)
        for (const Tensor &t : *tensors) {
            if (t.numel() == 0) continue;
            const Span s = span_of(t);
            const auto behind = std::lower_bound(spans.begin(), spans.end(), Span{s.second, 0});  // first that starts behind s
            TORCH_CHECK(behind == spans.begin() || std::prev(behind)->second <= s.first,
                        "Input mismatch: a gradient or the learning rate in the same memory as what the step writes");
        }
}

void adamw_step(const Tensors &params, const Tensors &grads, const Tensors &exp_avgs, const Tensors &exp_avg_sqs,
                const Tensor &steps, py::handle lr_, double beta1, double beta2, double eps, double weight_decay,
                const c10::optional<Tensors> &masters_, const c10::optional<Tensors> &m_scales_,
                const c10::optional<Tensors> &v_scales_, int64_t seed, int64_t first) {
    const size_t count = params.size();
    if (count == 0) return;
    const auto device = params[0].device();
    TORCH_CHECK(params[0].is_cuda(), "Input mismatch: parameters must be GPU (HIP) tensors");
    const auto param_dtype = same(params, {at::kFloat, at::kBFloat16}, params, "parameters");
    const auto grad_dtype = same(grads, {at::kFloat, at::kBFloat16}, params, "gradients");
    const auto state_dtype = same(exp_avgs, {at::kFloat, at::kFloat8_e4m3fn}, params, "states");
    same(exp_avg_sqs, {state_dtype}, params, "states");
    same_sizes(grads, params, "a gradient,");
    same_sizes(exp_avgs, params, "a state,");
    same_sizes(exp_avg_sqs, params, "a state,");
    const bool eight = state_dtype == at::kFloat8_e4m3fn;
    const Tensors none;
    const Tensors &masters = masters_ ? *masters_ : none, &m_scales = m_scales_ ? *m_scales_ : none,
                  &v_scales = v_scales_ ? *v_scales_ : none;
    if (eight) {
        TORCH_CHECK(m_scales_ && v_scales_, "Input mismatch: states in 8 bits need their scales");
        for (const Tensors *scales : {&m_scales, &v_scales}) {
            same(*scales, {at::kFloat8_e8m0fnu}, params, "scales");
            same_sizes(*scales, params, "a state's scales,", kBlock);
        }
    } else {
        TORCH_CHECK(!m_scales_ && !v_scales_, "Input mismatch: states in 32 bits have no scales");
    }
    if (param_dtype == at::kBFloat16) {
        TORCH_CHECK(masters_, "Input mismatch: bfloat16 parameters need their float32 masters");
        same(masters, {at::kFloat}, params, "masters");
        same_sizes(masters, params, "a master,");
    } else {
        TORCH_CHECK(!masters_, "Input mismatch: float32 parameters have no masters");
    }
    TORCH_CHECK(steps.device() == device && steps.scalar_type() == at::kInt && steps.dim() == 1 &&
                    steps.numel() == (int64_t)count && steps.is_contiguous(),
                "Input mismatch: steps must be contiguous int32 [parameters] on their device");
    double lr = 0.0;
    Tensor lr_tensor;
    if (THPVariable_Check(lr_.ptr())) {
        lr_tensor = THPVariable_Unpack(lr_.ptr());
        if (lr_tensor.device() == device) {
            TORCH_CHECK(lr_tensor.scalar_type() == at::kFloat && lr_tensor.numel() == 1,
                        "Input mismatch: a learning rate on the device must be a float32 scalar");
        } else {
            lr = lr_tensor.item<double>();
            lr_tensor = Tensor();
        }
    } else {
        lr = lr_.cast<double>();
    }
    const Tensors step_list = {steps};
    Tensors rate;
    if (lr_tensor.defined()) rate.push_back(lr_tensor);
    refuse_overlaps({&params, &exp_avgs, &exp_avg_sqs, &masters, &m_scales, &v_scales, &step_list}, {&grads, &rate});
    std::vector<gnnagg_adamw_tensor> records(count);
    for (size_t i = 0; i < count; ++i) {
        gnnagg_adamw_tensor &r = records[i];
        r.param = params[i].data_ptr();
        r.grad = grads[i].const_data_ptr();
        r.exp_avg = exp_avgs[i].data_ptr();
        r.exp_avg_sq = exp_avg_sqs[i].data_ptr();
        r.exp_avg_scales = eight ? bytes(m_scales[i]) : nullptr;
        r.exp_avg_sq_scales = eight ? bytes(v_scales[i]) : nullptr;
        r.master = masters_ ? masters[i].data_ptr<float>() : nullptr;
        r.n = params[i].numel();
    }
    const Place place(params[0]);
    check_rc(gnnagg_adamw_step(records.data(), (int64_t)count, steps.data_ptr<int32_t>(),
                               dtype_code(param_dtype, "parameters"), dtype_code(grad_dtype, "gradients"), eight ? 8 : 32, lr,
                               lr_tensor.defined() ? lr_tensor.const_data_ptr<float>() : nullptr, beta1, beta2, eps,
                               weight_decay, (uint32_t)seed, first, place.stream));
    for (const Tensors *tensors : {&params, &exp_avgs, &exp_avg_sqs, &masters, &m_scales, &v_scales})
        for (const Tensor &t : *tensors) changed(t);
    changed(steps);
}

}  // namespace

PYBIND11_MODULE(train_ops, m) {
    if (gnnagg_train_abi_version() != GNNAGG_TRAIN_ABI_VERSION)
        throw std::runtime_error("train_ops was compiled against libgnnagg training ABI version " +
                                 std::to_string(GNNAGG_TRAIN_ABI_VERSION) + " but the library it loaded reports " +
                                 std::to_string(gnnagg_train_abi_version()) +
                                 ": rebuild both (gnn_benchmark_amd/ext/build.sh)");
    m.doc() = "Calls of the training operators (libgnnagg.so underneath)";
    m.def("set_error_class", [](py::object cls) { error_class = cls.release().ptr(); });
    m.def("rms_norm", &differentiable_rms_norm);
    m.def("rms_norm_forward", &rms_norm);
    m.def("rms_norm_backward", &rms_norm_backward);
    m.def("rms_norm_fp8", &public_rms_norm_fp8);
    m.def("quantize_rows", &public_quantize_rows);
    m.def("quantize_weight", &public_quantize_weight);
    m.def("product", &public_product);
    m.def("weight_gradient", &public_weight_gradient);
    m.def("linear", &linear);
    m.def("norm_linear", &norm_linear);
    m.def("adamw_step", &adamw_step);
}
