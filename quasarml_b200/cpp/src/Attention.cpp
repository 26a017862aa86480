// The attention sublayer's operators over libqsml_cuda.so (see Ops/Attention.h).
#include "Ops/Attention.h"

#include <cmath>

#include "Common/Assert.h"

namespace QuasarML {
namespace Ops {

namespace {

using TP = std::shared_ptr<Tensor>;

// A descriptor argument that may be absent.
struct Arg {
    TP t;
    qsml_tdesc d;
    explicit Arg(TP tensor) : t(std::move(tensor)), d{} {
        if (t) d = t->desc();
    }
    const qsml_tdesc* get() const { return t ? &d : nullptr; }
};

// As it lies where its last dim has unit stride, else a copy.
TP in_place(const TP& t) {
    if (!t || t->rank() == 0 || t->dim(t->rank() - 1) <= 1 || t->strides().back() == 1) return t;
    return t->contiguous();
}
TP dense(const TP& t) { return t ? t->contiguous() : t; }

const int32_t* sections_of(const RotaryOptions& o) { return o.sections.empty() ? nullptr : o.sections.data(); }

float scale_of(const TP& q, const AttentionOptions& o) {
    if (o.scale != 0.0f) return o.scale;
    QS_ASSERT(q->rank() == 4 && q->dim(3) > 0, "attention needs [sequences, queries, heads, columns]");
    return 1.0f / std::sqrt(static_cast<float>(q->dim(3)));
}

}  // namespace

QueriesKeys norm_rotary(Device& d, TP q, TP k, TP wq, TP wk, TP positions, TP frequencies, const RotaryOptions& o) {
    QS_ASSERT(q && positions && frequencies, "null tensor");
    const Arg Q(in_place(q)), K(in_place(k)), WQ(dense(wq)), WK(dense(wk)), P(positions), F(dense(frequencies));
    QueriesKeys out{d.create_tensor(q->shape(), q->dtype()), k ? d.create_tensor(k->shape(), k->dtype()) : nullptr};
    const Arg OQ(out.q), OK(out.k);
    d.check(qsml_norm_rotary(d.ctx(), Q.get(), K.get(), WQ.get(), WK.get(), o.eps, P.get(), F.get(), sections_of(o),
                             static_cast<int32_t>(o.sections.size()), static_cast<int32_t>(o.pairing), OQ.get(), OK.get()));
    return out;
}

NormRotaryGrads norm_rotary_backward(Device& d, TP q, TP k, TP wq, TP wk, TP positions, TP frequencies, TP dq_out, TP dk_out,
                                     const RotaryOptions& o) {
    QS_ASSERT(q && positions && frequencies && dq_out, "null tensor");
    auto like = [&](const TP& t) { return t ? d.create_tensor(t->shape(), t->dtype()) : nullptr; };
    const Arg Q(in_place(q)), K(in_place(k)), WQ(dense(wq)), WK(dense(wk)), P(positions), F(dense(frequencies)),
        GQ(in_place(dq_out)), GK(in_place(dk_out));
    NormRotaryGrads g{like(q), like(k), like(wq), like(wk)};
    const Arg DQ(g.dq), DK(g.dk), DWQ(g.dwq), DWK(g.dwk);
    d.check(qsml_norm_rotary_backward(d.ctx(), Q.get(), K.get(), WQ.get(), WK.get(), o.eps, P.get(), F.get(), sections_of(o),
                                      static_cast<int32_t>(o.sections.size()), static_cast<int32_t>(o.pairing), GQ.get(),
                                      GK.get(), DQ.get(), DK.get(), DWQ.get(), DWK.get()));
    return g;
}

TP attention(Device& d, TP q, TP k, TP v, const AttentionOptions& o, TP* keep_lse) {
    QS_ASSERT(q && k && v, "null tensor");
    const float scale = scale_of(q, o);
    const Arg Q(in_place(q)), K(in_place(k)), V(in_place(v)), NQ(o.q_lengths), NK(o.k_lengths);
    const Arg O(d.create_tensor(q->shape(), q->dtype()));
    QS_ASSERT(!keep_lse || q->rank() == 4, "attention needs [sequences, queries, heads, columns]");
    const Arg L(keep_lse ? d.create_tensor({q->dim(0), q->dim(2), q->dim(1)}, DataType::F32) : nullptr);
    d.check(qsml_attention(d.ctx(), Q.get(), K.get(), V.get(), NQ.get(), NK.get(), scale, static_cast<int64_t>(o.window),
                           static_cast<int64_t>(o.sinks), L.get(), O.get()));
    if (keep_lse) *keep_lse = L.t;
    return O.t;
}

AttentionGrads attention_backward(Device& d, TP q, TP k, TP v, TP o, TP lse, TP dout, const AttentionOptions& opt) {
    QS_ASSERT(q && k && v && o && lse && dout, "null tensor");
    const float scale = scale_of(q, opt);
    const Arg Q(in_place(q)), K(in_place(k)), V(in_place(v)), O(in_place(o)), L(dense(lse)), G(in_place(dout)),
        NQ(opt.q_lengths), NK(opt.k_lengths);
    AttentionGrads g{d.create_tensor(q->shape(), q->dtype()), d.create_tensor(k->shape(), k->dtype()),
                     d.create_tensor(v->shape(), v->dtype())};
    const Arg DQ(g.dq), DK(g.dk), DV(g.dv);
    d.check(qsml_attention_backward(d.ctx(), Q.get(), K.get(), V.get(), O.get(), L.get(), G.get(), NQ.get(), NK.get(), scale,
                                    static_cast<int64_t>(opt.window), static_cast<int64_t>(opt.sinks), DQ.get(), DK.get(),
                                    DV.get()));
    return g;
}

}  // namespace Ops
}  // namespace QuasarML
