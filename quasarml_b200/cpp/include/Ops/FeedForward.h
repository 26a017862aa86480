// Linear and gated linear layers with their backward passes, and the layer
// norm's (additions of this backend; the reference has the product alone and no
// gradients).  Each is one call of the C ABI; a layer's bias, activation and
// residual run in its product's kernel.
#pragma once

#include <memory>

#include "../Core/Device.h"
#include "../Core/Tensor.h"

namespace QuasarML {

// Same codes as QSML_ACT_*.  Gelu is Ops::gelu's tanh form; Silu(z) = z * sigmoid(z).
enum class Activation : u32 { None = 0, Relu, Gelu, Silu, Sigmoid };

struct LayerNormGrads {
    std::shared_ptr<Tensor> dx, dgamma, dbeta;
};
struct LinearGrads {
    std::shared_ptr<Tensor> dx, dw, dbias;  // dbias null unless asked for
};
struct GatedLinearGrads {
    std::shared_ptr<Tensor> dx, dw_gate, dw_up, db_gate, db_up;  // db_* null unless asked for
};

namespace Ops {

// Gradients of layer_norm(x, gamma, beta, eps) from dy; dgamma and dbeta have gamma's dtype.
QS_API LayerNormGrads layer_norm_backward(Device& device, std::shared_ptr<Tensor> x, std::shared_ptr<Tensor> gamma,
                                          std::shared_ptr<Tensor> dy, f32 eps = 1e-5f);

// act(x w + bias) + residual; x [.., K], w [K, N] (any strides: a transposed view is read in place).
// bias and residual may be null.  keep: takes x w + bias for linear_backward.
QS_API std::shared_ptr<Tensor> linear(Device& device, std::shared_ptr<Tensor> x, std::shared_ptr<Tensor> w,
                                      std::shared_ptr<Tensor> bias = nullptr, Activation act = Activation::None,
                                      std::shared_ptr<Tensor> residual = nullptr, std::shared_ptr<Tensor>* keep = nullptr);
// pre: what linear kept (null without an activation).  dbias is F32.
QS_API LinearGrads linear_backward(Device& device, std::shared_ptr<Tensor> x, std::shared_ptr<Tensor> w, Activation act,
                                   std::shared_ptr<Tensor> pre, std::shared_ptr<Tensor> dy, bool want_dbias = false);

// act(x w_gate + b_gate) * (x w_up + b_up); keep_gate and keep_up take the two products.
QS_API std::shared_ptr<Tensor> gated_linear(Device& device, std::shared_ptr<Tensor> x, std::shared_ptr<Tensor> w_gate,
                                            std::shared_ptr<Tensor> w_up, Activation act = Activation::Silu,
                                            std::shared_ptr<Tensor> b_gate = nullptr, std::shared_ptr<Tensor> b_up = nullptr,
                                            std::shared_ptr<Tensor>* keep_gate = nullptr,
                                            std::shared_ptr<Tensor>* keep_up = nullptr);
QS_API GatedLinearGrads gated_linear_backward(Device& device, std::shared_ptr<Tensor> x, std::shared_ptr<Tensor> w_gate,
                                              std::shared_ptr<Tensor> w_up, Activation act, std::shared_ptr<Tensor> gate,
                                              std::shared_ptr<Tensor> up, std::shared_ptr<Tensor> dy,
                                              bool want_dbias = false);

}  // namespace Ops
}  // namespace QuasarML
