// Linear and gated linear layers, and the backward passes, over
// libqsml_cuda.so (see Ops/FeedForward.h).
#include "Ops/FeedForward.h"

#include "Common/Assert.h"

namespace QuasarML {
namespace Ops {

namespace {

using TP = std::shared_ptr<Tensor>;

// x with leading dims that fold into rows: a matrix as it lies, more dims contiguous.
TP rows_of(const TP& x) {
    QS_ASSERT(x && x->rank() >= 1, "a linear layer's input needs at least one dim");
    return x->rank() <= 2 ? x : x->contiguous();
}

std::vector<u32> with_last(const TP& x, const TP& w) {
    QS_ASSERT(w && w->rank() == 2, "a linear layer's weight needs two dims");
    auto shape = x->shape();
    shape.back() = w->dim(1);
    return shape;
}

// A descriptor argument that may be absent.
struct Arg {
    TP t;
    qsml_tdesc d;
    explicit Arg(TP tensor) : t(std::move(tensor)), d{} {
        if (t) d = t->desc();
    }
    const qsml_tdesc* get() const { return t ? &d : nullptr; }
};

TP dense(const TP& t) { return t ? t->contiguous() : t; }

}  // namespace

LayerNormGrads layer_norm_backward(Device& d, TP x, TP gamma, TP dy, f32 eps) {
    QS_ASSERT(x && gamma && dy, "null tensor");
    LayerNormGrads g{d.create_tensor(x->shape(), x->dtype()), d.create_tensor(gamma->shape(), gamma->dtype()),
                     d.create_tensor(gamma->shape(), gamma->dtype())};
    const Arg X(x->contiguous()), G(gamma->contiguous()), DY(dy->contiguous()), DX(g.dx), DG(g.dgamma), DB(g.dbeta);
    d.check(qsml_layer_norm_backward(d.ctx(), X.get(), G.get(), DY.get(), eps, DX.get(), DG.get(), DB.get()));
    return g;
}

TP linear(Device& d, TP x, TP w, TP bias, Activation act, TP residual, TP* keep) {
    const Arg X(rows_of(x)), W(w), B(dense(bias)), R(dense(residual));
    const auto shape = with_last(x, w);
    const Arg Y(d.create_tensor(shape, x->dtype())), P(keep ? d.create_tensor(shape, x->dtype()) : nullptr);
    d.check(qsml_linear(d.ctx(), X.get(), W.get(), B.get(), static_cast<int32_t>(act), R.get(), P.get(), Y.get(),
                        QSML_MM_AUTO));
    if (keep) *keep = P.t;
    return Y.t;
}

LinearGrads linear_backward(Device& d, TP x, TP w, Activation act, TP pre, TP dy, bool want_dbias) {
    QS_ASSERT(dy, "null tensor");
    const Arg X(rows_of(x)), W(w), P(dense(pre)), DY(dy->contiguous());
    with_last(x, w);
    LinearGrads g{d.create_tensor(x->shape(), x->dtype()), d.create_tensor(w->shape(), x->dtype()),
                  want_dbias ? d.create_tensor({w->dim(1)}, DataType::F32) : nullptr};
    const Arg DX(g.dx), DW(g.dw), DB(g.dbias);
    d.check(qsml_linear_backward(d.ctx(), X.get(), W.get(), static_cast<int32_t>(act), P.get(), DY.get(), DX.get(), DW.get(),
                                 DB.get(), QSML_MM_AUTO));
    return g;
}

TP gated_linear(Device& d, TP x, TP w_gate, TP w_up, Activation act, TP b_gate, TP b_up, TP* keep_gate, TP* keep_up) {
    const Arg X(rows_of(x)), WG(w_gate), WU(w_up), BG(dense(b_gate)), BU(dense(b_up));
    QS_ASSERT(w_up, "null tensor");
    const auto shape = with_last(x, w_gate);
    const Arg Y(d.create_tensor(shape, x->dtype())), G(keep_gate ? d.create_tensor(shape, x->dtype()) : nullptr),
        U(keep_up ? d.create_tensor(shape, x->dtype()) : nullptr);
    d.check(qsml_gated_linear(d.ctx(), X.get(), WG.get(), WU.get(), BG.get(), BU.get(), static_cast<int32_t>(act), G.get(),
                              U.get(), Y.get(), QSML_MM_AUTO));
    if (keep_gate) *keep_gate = G.t;
    if (keep_up) *keep_up = U.t;
    return Y.t;
}

GatedLinearGrads gated_linear_backward(Device& d, TP x, TP w_gate, TP w_up, Activation act, TP gate, TP up, TP dy,
                                       bool want_dbias) {
    QS_ASSERT(w_up && gate && up && dy, "null tensor");
    const Arg X(rows_of(x)), WG(w_gate), WU(w_up), G(gate->contiguous()), U(up->contiguous()), DY(dy->contiguous());
    with_last(x, w_gate);
    auto bias = [&]() { return want_dbias ? d.create_tensor({w_gate->dim(1)}, DataType::F32) : nullptr; };
    GatedLinearGrads g{d.create_tensor(x->shape(), x->dtype()), d.create_tensor(w_gate->shape(), x->dtype()),
                       d.create_tensor(w_up->shape(), x->dtype()), bias(), bias()};
    const Arg DX(g.dx), DG(g.dw_gate), DU(g.dw_up), BG(g.db_gate), BU(g.db_up);
    d.check(qsml_gated_linear_backward(d.ctx(), X.get(), WG.get(), WU.get(), static_cast<int32_t>(act), G.get(), U.get(),
                                       DY.get(), DX.get(), DG.get(), DU.get(), BG.get(), BU.get(), QSML_MM_AUTO));
    return g;
}

}  // namespace Ops
}  // namespace QuasarML
