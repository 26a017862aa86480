// qsml_attention and its backward pass: argument checks and the choice of kernels.
// The reference has no attention (its softmax, Ops/Elementwise.cpp:395-417, is a
// dispatch of its own over scores that a matmul would have written).
#include "attention.cuh"

namespace qsml {
namespace attn {
namespace {

using heads::Dims;
using heads::fail;
using heads::Named;

// A tensor of the sizes `like`.
qsml_status_t check_heads(Context* ctx, const char* op, Named t, int32_t dtype, const Dims& like, bool output, View* v) {
    if (!t.d) return QSML_OK;
    if (t.d->dtype != dtype) return fail(ctx, QSML_E_DTYPE, op, std::string(t.name) + " must have q's dtype");
    if (t.d->ndim != 4) return fail(ctx, QSML_E_SHAPE, op, std::string(t.name) + " must be [sequences, tokens, heads, columns]");
    Dims d;
    QSML_TRY_STATUS(heads::view_of(ctx, op, t, output, &d, v));
    if (d.B != like.B || d.S != like.S || d.H != like.H || d.D != like.D)
        return fail(ctx, QSML_E_SHAPE, op, std::string(t.name) + " has the wrong shape");
    return QSML_OK;
}

qsml_status_t check_lengths(Context* ctx, const char* op, Named t, int64_t B, const int** p, int64_t* step) {
    if (!t.d) return QSML_OK;
    QSML_TRY_STATUS(check_desc(ctx, t.d, t.name));
    if (t.d->dtype != QSML_I32) return fail(ctx, QSML_E_DTYPE, op, std::string(t.name) + " must be I32");
    if (t.d->ndim != 1 || t.d->shape[0] != B) return fail(ctx, QSML_E_SHAPE, op, std::string(t.name) + " must be [sequences]");
    *p = static_cast<const int*>(t.d->data);
    *step = t.d->stride[0];
    return QSML_OK;
}

// What both directions share.
qsml_status_t check_inputs(Context* ctx, const char* op, const qsml_tdesc* q, const qsml_tdesc* k, const qsml_tdesc* v,
                           const qsml_tdesc* q_lengths, const qsml_tdesc* k_lengths, float scale, int64_t window,
                           int64_t sinks, Problem* p, Dims* dq, Dims* dk) {
    const Named all[3] = {{q, "q"}, {k, "k"}, {v, "v"}};
    for (const Named& t : all) QSML_TRY_STATUS(check_desc(ctx, t.d, t.name));
    if (q->dtype != QSML_F32 && q->dtype != QSML_F16) return fail(ctx, QSML_E_DTYPE, op, "q must be F32 or F16");
    if (q->ndim != 4 || k->ndim != 4) return fail(ctx, QSML_E_SHAPE, op, "q and k must be [sequences, tokens, heads, columns]");
    *dq = Dims{q->shape[0], q->shape[1], q->shape[2], q->shape[3]};
    *dk = Dims{k->shape[0], k->shape[1], k->shape[2], k->shape[3]};
    if (dk->B != dq->B || dk->D != dq->D) return fail(ctx, QSML_E_SHAPE, op, "q and k must have the same sequences and columns");
    if (dq->H == 0 ? dk->H != 0 : dk->H == 0 || dq->H % dk->H)
        return fail(ctx, QSML_E_SHAPE, op, "the heads of q must be a multiple of k's");
    if (dq->D < 1) return fail(ctx, QSML_E_SHAPE, op, "the heads have no columns");
    if (dq->D > 256) return fail(ctx, QSML_E_UNSUPPORTED, op, "heads of more than 256 columns");
    const int64_t most = 1 << 30;
    if (dq->B > most || dq->S > most || dk->S > most || dq->H > most || dq->B * dq->H > most)
        return fail(ctx, QSML_E_UNSUPPORTED, op, "dimensions too large");
    QSML_TRY_STATUS(check_heads(ctx, op, all[0], q->dtype, *dq, false, &p->q));
    QSML_TRY_STATUS(check_heads(ctx, op, all[1], q->dtype, *dk, false, &p->k));
    QSML_TRY_STATUS(check_heads(ctx, op, all[2], q->dtype, *dk, false, &p->v));
    if (!(scale > 0.0f && scale < INFINITY)) return fail(ctx, QSML_E_INVALID, op, "scale must be positive and finite");
    if (window < 0 || sinks < 0) return fail(ctx, QSML_E_INVALID, op, "window and sinks must not be negative");
    QSML_TRY_STATUS((check_lengths(ctx, op, {q_lengths, "q_lengths"}, dq->B, &p->nq, &p->nq_step)));
    QSML_TRY_STATUS((check_lengths(ctx, op, {k_lengths, "k_lengths"}, dq->B, &p->nk, &p->nk_step)));
    p->B = static_cast<int>(dq->B);
    p->Sq = static_cast<int>(dq->S);
    p->Sk = static_cast<int>(dk->S);
    p->Hq = static_cast<int>(dq->H);
    p->Hk = static_cast<int>(dk->H);
    p->G = p->Hk ? p->Hq / p->Hk : 1;
    p->D = static_cast<int>(dq->D);
    p->scale = scale;
    // a window that no key is outside of hides none
    p->window = window >= dk->S ? 0 : static_cast<int>(window);
    p->sinks = static_cast<int>(sinks < dk->S ? sinks : dk->S);
    p->f16 = q->dtype == QSML_F16;
    return QSML_OK;
}

qsml_status_t check_lse(Context* ctx, const char* op, const qsml_tdesc* lse, const Dims& dq, float** p) {
    QSML_TRY_STATUS(check_desc(ctx, lse, "lse"));
    if (lse->dtype != QSML_F32) return fail(ctx, QSML_E_DTYPE, op, "lse must be F32");
    if (lse->ndim != 3 || lse->shape[0] != dq.B || lse->shape[1] != dq.H || lse->shape[2] != dq.S)
        return fail(ctx, QSML_E_SHAPE, op, "lse must be [sequences, heads, queries]");
    if (!is_contiguous(lse)) return fail(ctx, QSML_E_UNSUPPORTED, op, "lse must be contiguous");
    *p = static_cast<float*>(lse->data);
    return QSML_OK;
}

// delta[b, h, i] = sum of dout * o over the columns: a warp a row.
template <typename T>
__global__ void __launch_bounds__(256) k_attention_delta(const __grid_constant__ Problem p, float* delta, int64_t rows) {
    pdl_begin();
    const int lane = threadIdx.x & 31;
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    if (row >= rows) return;
    const int i = static_cast<int>(row % p.Sq), h = static_cast<int>(row / p.Sq % p.Hq), b = static_cast<int>(row / p.Sq / p.Hq);
    float s = 0.0f;
    if (i < Seq(p, b).nq) {
        const T* x = reinterpret_cast<const T*>(p.o.p) + b * p.o.b + i * p.o.s + h * p.o.h;
        const T* y = reinterpret_cast<const T*>(p.dout.p) + b * p.dout.b + i * p.dout.s + h * p.dout.h;
        for (int c = lane; c < p.D; c += 32) s = fmaf(heads::to_f(x[c]), heads::to_f(y[c]), s);
    }
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    if (lane == 0) delta[row] = s;
}

qsml_status_t run_delta(Context* ctx, const Problem& p, float* delta) {
    const int64_t rows = static_cast<int64_t>(p.B) * p.Hq * p.Sq;
    const int64_t grid = (rows + 7) / 8;
    if (grid > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "qsml_attention_backward: dimensions too large");
    const cudaError_t e = launch_pdl(p.f16 ? k_attention_delta<__half> : k_attention_delta<float>, dim3(static_cast<unsigned>(grid)),
                                     dim3(256), 0, ctx->stream, p, delta, rows);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_attention_delta");
    return after_launch(ctx, "k_attention_delta");
}

}  // namespace
}  // namespace attn
}  // namespace qsml

using namespace qsml;
using namespace qsml::attn;

extern "C" qsml_status_t qsml_attention(qsml_ctx* handle, const qsml_tdesc* q, const qsml_tdesc* k, const qsml_tdesc* v,
                                        const qsml_tdesc* q_lengths, const qsml_tdesc* k_lengths, float scale, int64_t window,
                                        int64_t sinks, const qsml_tdesc* lse, const qsml_tdesc* o) try {
    QSML_CTX(handle);
    const char* op = "qsml_attention";
    Problem p;
    Dims dq, dk;
    QSML_TRY_STATUS(check_inputs(C_, op, q, k, v, q_lengths, k_lengths, scale, window, sinks, &p, &dq, &dk));
    QSML_TRY_STATUS(check_desc(C_, o, "o"));
    QSML_TRY_STATUS((check_heads(C_, op, {o, "o"}, q->dtype, dq, true, &p.o)));
    if (lse) QSML_TRY_STATUS(check_lse(C_, op, lse, dq, &p.lse));
    const Named in[5] = {{q, "q"}, {k, "k"}, {v, "v"}, {q_lengths, "q_lengths"}, {k_lengths, "k_lengths"}};
    const Named out[2] = {{o, "o"}, {lse, "lse"}};
    QSML_TRY_STATUS(heads::check_overlap(C_, op, in, 5, out, 2));
    if (numel(q) == 0) return QSML_OK;
    if (few_queries(p)) return forward_few(C_, p);
    return tc_takes(p) ? forward_tc(C_, p) : forward_simt(C_, p);
} QSML_NO_THROW

extern "C" qsml_status_t qsml_attention_backward(qsml_ctx* handle, const qsml_tdesc* q, const qsml_tdesc* k, const qsml_tdesc* v,
                                                 const qsml_tdesc* o, const qsml_tdesc* lse, const qsml_tdesc* dout,
                                                 const qsml_tdesc* q_lengths, const qsml_tdesc* k_lengths, float scale,
                                                 int64_t window, int64_t sinks, const qsml_tdesc* dq, const qsml_tdesc* dk,
                                                 const qsml_tdesc* dv) try {
    QSML_CTX(handle);
    const char* op = "qsml_attention_backward";
    Problem p;
    Dims nq, nk;
    QSML_TRY_STATUS(check_inputs(C_, op, q, k, v, q_lengths, k_lengths, scale, window, sinks, &p, &nq, &nk));
    QSML_TRY_STATUS(check_desc(C_, o, "o"));
    QSML_TRY_STATUS(check_desc(C_, dout, "dout"));
    QSML_TRY_STATUS(check_lse(C_, op, lse, nq, &p.lse));
    QSML_TRY_STATUS((check_heads(C_, op, {o, "o"}, q->dtype, nq, false, &p.o)));
    QSML_TRY_STATUS((check_heads(C_, op, {dout, "dout"}, q->dtype, nq, false, &p.dout)));
    const Named out[3] = {{dq, "dq"}, {dk, "dk"}, {dv, "dv"}};
    View* to[3] = {&p.dq, &p.dk, &p.dv};
    for (int i = 0; i < 3; ++i) {
        if (!out[i].d) continue;
        QSML_TRY_STATUS(check_desc(C_, out[i].d, out[i].name));
        QSML_TRY_STATUS(check_heads(C_, op, out[i], q->dtype, i ? nk : nq, true, to[i]));
    }
    const Named in[8] = {{q, "q"}, {k, "k"}, {v, "v"}, {o, "o"}, {lse, "lse"}, {dout, "dout"}, {q_lengths, "q_lengths"}, {k_lengths, "k_lengths"}};
    QSML_TRY_STATUS(heads::check_overlap(C_, op, in, 8, out, 3));
    if (numel(q) == 0) p.dq.p = nullptr;
    if (numel(k) == 0) p.dk.p = p.dv.p = nullptr;
    if (!p.dq.p && !p.dk.p && !p.dv.p) return QSML_OK;
    if (tc_takes_backward(p)) return backward_tc(C_, p);
    Workspace ws(C_);
    void* delta = nullptr;
    QSML_TRY_STATUS(ws.get(sizeof(float) * p.B * p.Hq * static_cast<size_t>(p.Sq), &delta));
    if (numel(q) && (p.dq.p || p.dk.p)) QSML_TRY_STATUS(run_delta(C_, p, static_cast<float*>(delta)));
    return backward_simt(C_, p, static_cast<const float*>(delta));
} QSML_NO_THROW
