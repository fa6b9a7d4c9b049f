// Decoding in 8 bits: rows as int8 with a scale each, products of them, and the token at the end.  None of it has a counterpart in Axiom; names and
// checks follow ops:: and nn::.  Everything runs when called (like ops::argmax), on the materialised inputs, and needs Device::GPU.
#pragma once

#include <string>

#include "axiom/nn.hpp"
#include "axiom/tensor.hpp"

namespace axiom {
namespace ops {

// values Int8 (..., n), scales Float32 (...): values * scales stands for the rows
struct Quantized {
    Tensor values, scales;
};

// Rows along the last dimension, scale = max |x| / 127, the nearest integers (halves to even).  A weight (out_features, in_features) by output channel,
// activations by token.  A row with an infinity or a NaN: scale NaN.
Quantized quantize_int8(const Tensor &x);

struct QuantizedNorm {
    Quantized normalized;
    Tensor sum; // x + residual, in x's type; empty without a residual
};
// ops::rms_norm(x + residual, weight) over the last dimension, quantized without being rounded in between.  residual and weight may be empty
// tensors; both have x's type, residual x's shape, weight (n).
QuantizedNorm rms_norm_int8(const Tensor &x, const Tensor &residual, const Tensor &weight, float eps = 1e-5f);

// activation(x W^T + bias + residual) in `dtype` (Float32, Float16, BFloat16; bias and residual are of it, or empty): x (..., k), weight (n, k).
// activation: "none", "relu", "gelu", "silu", "sigmoid" or "tanh".
Tensor linear_int8(const Quantized &x, const Quantized &weight, const Tensor &bias, const Tensor &residual, const std::string &activation, DType dtype);
Tensor linear_int8(const Quantized &x, const Quantized &weight, DType dtype);

// A setting for each row of logits (as many elements as there are rows), or an empty tensor: off.  temperature, top_p, min_p Float32, top_k Int32.
struct SampleSettings {
    Tensor temperature, top_k, top_p, min_p;
};
struct Sampled {
    Tensor tokens;        // Int64, logits' shape without the last dimension; -1 where a row has nothing to draw
    Tensor probabilities; // Float32, of the tokens among those that the filters keep
};
// Tokens by given random numbers u in [0, 1) (Float32, one for each row): see axhip_sample for what the settings keep and which token u falls on.
Sampled sample(const Tensor &logits, const Tensor &u, const SampleSettings &settings);
// the same settings for every row (they go with the launch: nothing is copied or waited for): temperature 0 is greedy; top_k 0, top_p 1 and min_p 0 are off
Sampled sample(const Tensor &logits, const Tensor &u, float temperature = 1.0f, int top_k = 0, float top_p = 1.0f, float min_p = 0.0f);

} // namespace ops

namespace nn {

// nn::Linear with its weight in 8 bits by output channel; inputs are quantized by token.  Parameters: weight Int8 (out_features, in_features),
// weight_scale Float32 (out_features), bias.
class QuantizedLinear : public Module {
  public:
    explicit QuantizedLinear(bool bias = true);
    explicit QuantizedLinear(const Linear &linear); // quantizes its weight (on the GPU)
    Tensor forward(const Tensor &input) const override; // result in the input's type
    // an input that is quantized already (ops::rms_norm_int8), a residual (or an empty tensor) and an activation
    Tensor forward(const ops::Quantized &input, DType dtype, const Tensor &residual, const std::string &activation = "none") const;
    Module &to(DType dtype) override; // the bias alone
    using Module::to;
    bool has_bias() const { return has_bias_; }
    const Tensor &weight() const { return weight_; }
    const Tensor &weight_scale() const { return weight_scale_; }
    const Tensor &bias() const { return bias_; }

  private:
    Tensor weight_, weight_scale_, bias_;
    bool has_bias_;
};

} // namespace nn
} // namespace axiom
