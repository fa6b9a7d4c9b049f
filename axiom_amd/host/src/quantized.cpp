// Rows in 8 bits, products of them and sampling over the C ABI.
#include "axiom/quantized.hpp"

#include "axiom/operations.hpp"
#include "hip_call.hpp"

namespace axiom::ops {
namespace {
void need_gpu(const char *who, const Tensor &t) {
    if (t.empty()) throw ValueError(std::string(who) + ": an empty tensor");
    if (t.device() != Device::GPU) throw RuntimeError(std::string("ops::") + who + " on CPU tensors: this library is the gfx950 GPU backend only; move the operands with .gpu()");
}
void need_floating(const char *who, const Tensor &t) {
    if (t.dtype() != DType::Float32 && t.dtype() != DType::Float16 && t.dtype() != DType::BFloat16) throw TypeError(std::string(who) + ": Float32, Float16 or BFloat16; got " + dtype_name(t.dtype()));
}
void need_type(const char *who, const char *what, const Tensor &t, DType want) {
    if (t.dtype() != want) throw TypeError(std::string(who) + ": " + what + " must be " + dtype_name(want) + ", got " + dtype_name(t.dtype()));
}
Shape without_last(const Shape &s) { return Shape(s.begin(), s.end() - 1); }
// contiguous, materialised
Tensor settled(const Tensor &t) {
    Tensor c = t.ascontiguousarray();
    c.sync();
    return c.ascontiguousarray();
}
const char *at(const Tensor &t) { return t.empty() ? nullptr : static_cast<const char *>(t.storage()->raw()) + t.offset(); }
char *out_at(const Tensor &t) { return static_cast<char *>(t.storage()->raw()); }

AxhipRowsQ8Params rows_of(const char *who, const Tensor &x) {
    if (x.ndim() == 0) throw ShapeError(std::string(who) + ": rows of a rank-0 tensor");
    AxhipRowsQ8Params p{};
    p.dtype = ::axiom::detail::to_axhip_dtype(x.dtype());
    p.cols = static_cast<int64_t>(x.shape().back());
    p.rows = static_cast<int64_t>(ShapeUtils::size(without_last(x.shape())));
    p.ld_x = p.ld_residual = p.ld_sum = p.ld_q = p.cols;
    return p;
}
Quantized room_for(const Tensor &x) { return {Tensor(x.shape(), DType::Int8, Device::GPU), Tensor(without_last(x.shape()), DType::Float32, Device::GPU)}; }
} // namespace

Quantized quantize_int8(const Tensor &x) {
    need_gpu("quantize_int8", x);
    need_floating("quantize_int8", x);
    const AxhipRowsQ8Params p = rows_of("quantize_int8", x);
    const Tensor src = settled(x);
    Quantized q = room_for(x);
    AXHIP_CALL(axhip_quantize_q8(at(src), reinterpret_cast<int8_t *>(out_at(q.values)), reinterpret_cast<float *>(out_at(q.scales)), &p, nullptr));
    return q; // asynchronous; .cpu() / item() synchronise
}

QuantizedNorm rms_norm_int8(const Tensor &x, const Tensor &residual, const Tensor &weight, float eps) {
    need_gpu("rms_norm_int8", x);
    need_floating("rms_norm_int8", x);
    AxhipRowsQ8Params p = rows_of("rms_norm_int8", x);
    p.eps = eps;
    if (!(eps >= 0.0f) || eps > 3.4e38f) throw ValueError("rms_norm_int8: eps must be a finite number, not negative");
    for (const Tensor *t : {&residual, &weight}) {
        if (t->empty()) continue;
        need_gpu("rms_norm_int8", *t);
        need_type("rms_norm_int8", t == &residual ? "residual" : "weight", *t, x.dtype());
    }
    if (!residual.empty() && residual.shape() != x.shape()) throw ShapeError("rms_norm_int8: residual must have the input's shape");
    if (!weight.empty() && (weight.ndim() != 1 || weight.shape()[0] != x.shape().back()))
        throw ShapeError("rms_norm_int8: weight must have shape [" + std::to_string(x.shape().back()) + "]");
    const Tensor src = settled(x), res = residual.empty() ? Tensor() : settled(residual), w = weight.empty() ? Tensor() : settled(weight);
    QuantizedNorm out{room_for(x), Tensor()};
    if (!residual.empty()) out.sum = Tensor(x.shape(), x.dtype(), Device::GPU);
    AXHIP_CALL(axhip_rms_norm_q8(at(src), at(res), at(w), residual.empty() ? nullptr : out_at(out.sum), reinterpret_cast<int8_t *>(out_at(out.normalized.values)),
                                 reinterpret_cast<float *>(out_at(out.normalized.scales)), &p, nullptr));
    return out;
}

Tensor linear_int8(const Quantized &x, const Quantized &weight, const Tensor &bias, const Tensor &residual, const std::string &activation, DType dtype) {
    const char *who = "linear_int8";
    for (const Tensor *t : {&x.values, &x.scales, &weight.values, &weight.scales}) need_gpu(who, *t);
    need_type(who, "values", x.values, DType::Int8);
    need_type(who, "values", weight.values, DType::Int8);
    need_type(who, "scales", x.scales, DType::Float32);
    need_type(who, "scales", weight.scales, DType::Float32);
    if (dtype != DType::Float32 && dtype != DType::Float16 && dtype != DType::BFloat16) throw TypeError("linear_int8: results are Float32, Float16 or BFloat16; got " + dtype_name(dtype));
    const Shape &xs = x.values.shape(), &ws = weight.values.shape();
    if (xs.empty() || ws.size() != 2 || xs.back() != ws[1]) throw ShapeError("linear_int8: input (..., k) and weight (n, k)");
    if (x.scales.shape() != without_last(xs) || weight.scales.shape() != without_last(ws)) throw ShapeError("linear_int8: a scale for each row of the input and of the weight");
    Shape out_shape = xs;
    out_shape.back() = ws[0];
    if (!bias.empty()) {
        need_gpu(who, bias);
        need_type(who, "bias", bias, dtype);
        if (bias.ndim() != 1 || bias.shape()[0] != ws[0]) throw ShapeError("linear_int8: bias must have shape [" + std::to_string(ws[0]) + "]");
    }
    if (!residual.empty()) {
        need_gpu(who, residual);
        need_type(who, "residual", residual, dtype);
        if (residual.shape() != out_shape) throw ShapeError("linear_int8: residual must have the result's shape");
    }
    AxhipGemmQ8Params p{};
    if (activation == "relu") p.epilogue_op = AXHIP_OP_RELU;
    else if (activation == "gelu") p.epilogue_op = AXHIP_OP_GELU;
    else if (activation == "silu") p.epilogue_op = AXHIP_OP_SILU;
    else if (activation == "sigmoid") p.epilogue_op = AXHIP_OP_SIGMOID;
    else if (activation == "tanh") p.epilogue_op = AXHIP_OP_TANH;
    else if (activation != "none") throw ValueError("linear_int8: activation must be 'none', 'relu', 'gelu', 'silu', 'sigmoid' or 'tanh', got '" + activation + "'");
    const Tensor a = settled(x.values), sa = settled(x.scales), b = settled(weight.values), sb = settled(weight.scales);
    const Tensor bi = bias.empty() ? Tensor() : settled(bias), res = residual.empty() ? Tensor() : settled(residual);
    p.dtype = ::axiom::detail::to_axhip_dtype(dtype);
    p.m = static_cast<int64_t>(ShapeUtils::size(without_last(xs)));
    p.n = static_cast<int64_t>(ws[0]);
    p.k = p.lda = p.ldb = static_cast<int64_t>(ws[1]);
    p.ldc = p.n;
    p.scale_a = reinterpret_cast<const float *>(at(sa));
    p.scale_b = reinterpret_cast<const float *>(at(sb));
    p.bias = at(bi);
    p.residual = at(res);
    Tensor out(out_shape, dtype, Device::GPU);
    AXHIP_CALL(axhip_gemm_q8(reinterpret_cast<const int8_t *>(at(a)), reinterpret_cast<const int8_t *>(at(b)), out_at(out), &p, nullptr));
    return out;
}
Tensor linear_int8(const Quantized &x, const Quantized &weight, DType dtype) { return linear_int8(x, weight, Tensor(), Tensor(), "none", dtype); }

namespace {
// The checks of both forms; `settings` puts the settings of so many rows into the parameters and keeps the tensors they lie in.
template <class F> Sampled draw(const Tensor &logits, const Tensor &u, F settings) {
    const char *who = "sample";
    need_gpu(who, logits);
    need_floating(who, logits);
    if (logits.ndim() == 0 || logits.shape().back() == 0) throw ShapeError("sample: logits (..., vocabulary)");
    const Shape out_shape = without_last(logits.shape());
    const size_t rows = ShapeUtils::size(out_shape);
    auto of_rows = [&](const char *what, const Tensor &t, DType want) {
        if (t.empty()) return Tensor();
        need_gpu(who, t);
        need_type(who, what, t, want);
        if (t.size() != rows) throw ShapeError(std::string("sample: ") + what + " needs a value for each of " + std::to_string(rows) + " rows, got " + std::to_string(t.size()));
        return settled(t);
    };
    if (u.empty()) throw ValueError("sample: a random number for each row");
    const Tensor src = settled(logits), un = of_rows("u", u, DType::Float32);
    AxhipSampleParams p{};
    p.dtype = ::axiom::detail::to_axhip_dtype(src.dtype());
    p.rows = static_cast<int64_t>(rows);
    p.vocab = p.ld = static_cast<int64_t>(logits.shape().back());
    p.u = reinterpret_cast<const float *>(at(un));
    [[maybe_unused]] const auto kept = settings(p, of_rows);
    Sampled out{Tensor(out_shape, DType::Int64, Device::GPU), Tensor(out_shape, DType::Float32, Device::GPU)};
    AXHIP_CALL(axhip_sample(at(src), reinterpret_cast<int64_t *>(out_at(out.tokens)), reinterpret_cast<float *>(out_at(out.probabilities)), &p, nullptr));
    return out;
}
} // namespace

Sampled sample(const Tensor &logits, const Tensor &u, const SampleSettings &settings) {
    return draw(logits, u, [&](AxhipSampleParams &p, auto of_rows) {
        SampleSettings s{of_rows("temperature", settings.temperature, DType::Float32), of_rows("top_k", settings.top_k, DType::Int32), of_rows("top_p", settings.top_p, DType::Float32),
                         of_rows("min_p", settings.min_p, DType::Float32)};
        p.temperature = reinterpret_cast<const float *>(at(s.temperature));
        p.top_k = reinterpret_cast<const int32_t *>(at(s.top_k));
        p.top_p = reinterpret_cast<const float *>(at(s.top_p));
        p.min_p = reinterpret_cast<const float *>(at(s.min_p));
        return s;
    });
}

Sampled sample(const Tensor &logits, const Tensor &u, float temperature, int top_k, float top_p, float min_p) {
    return draw(logits, u, [&](AxhipSampleParams &p, auto) {
        p.uniform = 1;
        p.all_temperature = temperature;
        p.all_top_k = top_k;
        p.all_top_p = top_p;
        p.all_min_p = min_p;
        return 0;
    });
}

} // namespace axiom::ops

namespace axiom::nn {

QuantizedLinear::QuantizedLinear(bool bias) : has_bias_(bias) {
    register_parameter("weight", weight_);
    register_parameter("weight_scale", weight_scale_);
    if (bias) register_parameter("bias", bias_);
}

QuantizedLinear::QuantizedLinear(const Linear &linear) : QuantizedLinear(linear.has_bias()) {
    if (linear.weight().empty()) throw RuntimeError("QuantizedLinear: the Linear's weight is not initialized (load_state_dict first)");
    ops::Quantized q = ops::quantize_int8(linear.weight());
    weight_ = q.values;
    weight_scale_ = q.scales;
    if (has_bias_) bias_ = linear.bias();
    if (!bias_.empty() && bias_.is_lazy()) bias_.sync();
}

Tensor QuantizedLinear::forward(const Tensor &input) const { return forward(ops::quantize_int8(input), input.dtype(), Tensor()); }

Tensor QuantizedLinear::forward(const ops::Quantized &input, DType dtype, const Tensor &residual, const std::string &activation) const {
    if (weight_.empty()) throw RuntimeError("QuantizedLinear: weight not initialized (load_state_dict first)");
    Tensor bias = has_bias_ ? bias_ : Tensor();
    if (!bias.empty() && bias.dtype() != dtype) bias = bias.astype(dtype);
    return ops::linear_int8(input, {weight_, weight_scale_}, bias, residual, activation, dtype);
}

Module &QuantizedLinear::to(DType dtype) {
    if (!bias_.empty()) {
        bias_ = bias_.astype(dtype);
        bias_.sync();
    }
    return *this;
}

} // namespace axiom::nn
