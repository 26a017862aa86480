// qsml_linear, qsml_gated_linear and their backward passes: argument checks and
// the choice of kernels.
//
// The reference has the product alone (Ops::matmul, Ops/LinAlg.cpp:221-271),
// every further step of a layer being a dispatch that reads and writes the
// whole result (Ops/Elementwise.cpp:139-417), and no gradients.
#include "linear.cuh"
#include "linear_grad.cuh"

namespace qsml {
namespace linear {
namespace {

struct Named {
    const qsml_tdesc* d;
    const char* name;
};

qsml_status_t fail(Context* ctx, qsml_status_t st, const char* op, const std::string& what) {
    return set_error(ctx, st, std::string(op) + ": " + what);
}

// The leading dims of d as one: rows and the elements between them.  False if
// their strides do not chain.
bool rows_of(const qsml_tdesc* d, int64_t* rows, int64_t* rs) {
    *rows = 1;
    *rs = 0;
    for (int i = d->ndim - 2; i >= 0; --i) {
        if (d->shape[i] == 1) continue;
        if (d->shape[i] == 0) {
            *rows = 0;
            return true;
        }
        if (*rows > 1 && d->stride[i] != *rs * *rows) return false;
        if (*rows == 1) *rs = d->stride[i];
        *rows *= d->shape[i];
    }
    return true;
}

qsml_status_t matrix_of(Context* ctx, const char* op, Named x, Mat* m) {
    if (x.d->ndim < 1) return fail(ctx, QSML_E_SHAPE, op, std::string(x.name) + " needs at least one dim");
    m->p = x.d->data;
    m->cols = x.d->shape[x.d->ndim - 1];
    m->cs = x.d->stride[x.d->ndim - 1];
    if (!rows_of(x.d, &m->rows, &m->rs))
        return fail(ctx, QSML_E_UNSUPPORTED, op, std::string("the leading dims of ") + x.name +
                                                     " do not fold into rows of one stride (materialise with qsml_gather)");
    return QSML_OK;
}

// d has the leading dims of `like` and `last` as its last one.
bool shaped(const qsml_tdesc* d, const qsml_tdesc* like, int64_t last) {
    if (d->ndim != like->ndim || d->shape[d->ndim - 1] != last) return false;
    for (int i = 0; i + 1 < d->ndim; ++i)
        if (d->shape[i] != like->shape[i]) return false;
    return true;
}

bool same_view(const qsml_tdesc* a, const qsml_tdesc* b) {
    if (a->data != b->data || a->dtype != b->dtype || a->ndim != b->ndim) return false;
    for (int i = 0; i < a->ndim; ++i)
        if (a->shape[i] != b->shape[i] || (a->shape[i] > 1 && a->stride[i] != b->stride[i])) return false;
    return true;
}

// No output may meet an input or another output; `inplace` may be read where
// `out0` is written, element for element.
qsml_status_t check_overlap(Context* ctx, const char* op, const Named* in, int ni, const Named* out, int no,
                            const qsml_tdesc* inplace) {
    for (int o = 0; o < no; ++o) {
        if (!out[o].d) continue;
        for (int i = 0; i < ni; ++i) {
            if (!in[i].d || !views_meet(out[o].d, in[i].d)) continue;
            if (o == 0 && in[i].d == inplace && same_view(in[i].d, out[o].d)) continue;
            return fail(ctx, QSML_E_INVALID, op, std::string(out[o].name) + " overlaps " + in[i].name);
        }
        for (int i = 0; i < o; ++i)
            if (out[i].d && views_meet(out[o].d, out[i].d))
                return fail(ctx, QSML_E_INVALID, op, std::string(out[o].name) + " overlaps " + out[i].name);
    }
    return QSML_OK;
}

qsml_status_t check_all(Context* ctx, const Named* t, int n, int required) {
    for (int i = 0; i < n; ++i)
        if (i < required || t[i].d) QSML_TRY_STATUS(check_desc(ctx, t[i].d, t[i].name));
    return QSML_OK;
}

qsml_status_t check_act(Context* ctx, const char* op, int32_t act) {
    if (act < QSML_ACT_NONE || act > QSML_ACT_SIGMOID) return fail(ctx, QSML_E_INVALID, op, "unknown activation");
    return QSML_OK;
}

qsml_status_t check_precision(Context* ctx, const char* op, int32_t dtype, int32_t precision) {
    if (dtype != QSML_F32 && dtype != QSML_F16) return fail(ctx, QSML_E_DTYPE, op, "x must be F32 or F16");
    const bool ok = precision == QSML_MM_AUTO ||
                    (dtype == QSML_F32 ? precision == QSML_MM_FP32_FFMA : precision == QSML_MM_FP16_F32ACC);
    if (!ok) return fail(ctx, QSML_E_INVALID, op, "precision does not apply to this dtype");
    return QSML_OK;
}

// x [.., K] and w [K, N] (w2 alike) to the sizes and matrices of a problem.
qsml_status_t check_xw(Context* ctx, const char* op, const qsml_tdesc* x, const qsml_tdesc* const* w, const char* const* names,
                       int nw, Mat* mx, Mat* mw) {
    QSML_TRY_STATUS(matrix_of(ctx, op, Named{x, "x"}, mx));
    for (int i = 0; i < nw; ++i) {
        if (w[i]->dtype != x->dtype) return fail(ctx, QSML_E_DTYPE, op, std::string(names[i]) + " must have x's dtype");
        if (w[i]->ndim != 2 || w[i]->shape[0] != mx->cols || (i && w[i]->shape[1] != w[0]->shape[1]))
            return fail(ctx, QSML_E_SHAPE, op, std::string(names[i]) + " must be [x's last dim, features]");
        QSML_TRY_STATUS(matrix_of(ctx, op, Named{w[i], names[i]}, &mw[i]));
        mw[i].rs = w[i]->stride[0];
        mw[i].rows = w[i]->shape[0];
    }
    if (mx->rows > INT32_MAX || mx->cols > INT32_MAX || mw[0].cols > INT32_MAX)
        return fail(ctx, QSML_E_UNSUPPORTED, op, "dimensions too large");
    return QSML_OK;
}

// A [N] parameter or its gradient: contiguous, F32 or x's dtype.
qsml_status_t check_vector(Context* ctx, const char* op, Named v, int32_t dtype, int64_t n) {
    if (!v.d) return QSML_OK;
    if (v.d->dtype != QSML_F32 && v.d->dtype != dtype)
        return fail(ctx, QSML_E_DTYPE, op, std::string(v.name) + " must be F32 or x's dtype");
    if (v.d->ndim != 1 || v.d->shape[0] != n) return fail(ctx, QSML_E_SHAPE, op, std::string(v.name) + " must be [features]");
    if (!is_contiguous(v.d)) return fail(ctx, QSML_E_UNSUPPORTED, op, std::string(v.name) + " must be contiguous");
    return QSML_OK;
}

// A tensor of x's leading dims and `last`, of x's dtype; contiguous unless `ld`
// is given, which then takes the elements between its rows.
qsml_status_t check_rows(Context* ctx, const char* op, Named v, const qsml_tdesc* x, int64_t last, int64_t* ld = nullptr) {
    if (!v.d) return QSML_OK;
    if (v.d->dtype != x->dtype) return fail(ctx, QSML_E_DTYPE, op, std::string(v.name) + " must have x's dtype");
    if (!shaped(v.d, x, last)) return fail(ctx, QSML_E_SHAPE, op, std::string(v.name) + " has the wrong shape");
    if (!ld) {
        if (!is_contiguous(v.d)) return fail(ctx, QSML_E_UNSUPPORTED, op, std::string(v.name) + " must be contiguous");
        return QSML_OK;
    }
    int64_t rows;
    if (numel(v.d) == 0) {  // no element is addressed
        *ld = 0;
        return QSML_OK;
    }
    if (!rows_of(v.d, &rows, ld) || (last > 1 && v.d->stride[v.d->ndim - 1] != 1))
        return fail(ctx, QSML_E_UNSUPPORTED, op, std::string(v.name) + " needs unit stride in its last dim and rows of one stride");
    return QSML_OK;
}

// The gradient of a weight: [K, N], contiguous, x's dtype.
qsml_status_t check_dw(Context* ctx, const char* op, Named v, int32_t dtype, int64_t K, int64_t N) {
    if (!v.d) return QSML_OK;
    if (v.d->dtype != dtype) return fail(ctx, QSML_E_DTYPE, op, std::string(v.name) + " must have x's dtype");
    if (v.d->ndim != 2 || v.d->shape[0] != K || v.d->shape[1] != N)
        return fail(ctx, QSML_E_SHAPE, op, std::string(v.name) + " must have w's shape");
    if (!is_contiguous(v.d)) return fail(ctx, QSML_E_UNSUPPORTED, op, std::string(v.name) + " must be contiguous");
    return QSML_OK;
}

void set_vec(Epilogue* e, int es) {
    // the biases are read as single elements where not all is whole
    const void* p[6] = {e->residual, e->pre[0], e->pre[1], e->y, e->bias[0], e->bias[1]};
    auto aligned = [&](int n, int64_t elements) {
        bool v = e->N % elements == 0;
        for (int i = 0; i < n; ++i) v = v && reinterpret_cast<uintptr_t>(p[i]) % (n == 6 ? 16 : elements * es) == 0;
        return v && (!e->residual || e->res_ld % elements == 0);
    };
    e->vec = aligned(6, 8) ? 1 : aligned(4, 2) ? 2 : 0;
}

bool on_tensor_cores(int32_t precision, const Problem& p) { return precision != QSML_MM_FP32_FFMA && p.K > 0; }

// The products of n problems (at most 2), by the kernels that take them.
qsml_status_t run(Context* ctx, int32_t dtype, int32_t precision, Problem* const* all, int n) {
    const Problem* tc[2];
    int ntc = 0;
    for (int i = 0; i < n; ++i) {
        Problem& p = *all[i];
        if (p.M == 0 || p.N == 0) continue;
        if (!p.e.y && !p.e.pre[0] && !p.e.pre[1]) continue;
        p.e.N = p.N;
        set_vec(&p.e, dtype_size(dtype));
        if (dtype == QSML_F32 && few_rows(p))
            QSML_TRY_STATUS(run_few(ctx, p));
        else if (on_tensor_cores(precision, p))
            tc[ntc++] = &p;
        else
            QSML_TRY_STATUS(dtype == QSML_F32 ? run_simt<float>(ctx, p) : run_simt<__half>(ctx, p));
    }
    return ntc ? run_tc(ctx, tc, ntc, dtype == QSML_F32) : QSML_OK;
}
qsml_status_t run(Context* ctx, int32_t dtype, int32_t precision, Problem& p) {
    Problem* one = &p;
    return run(ctx, dtype, precision, &one, 1);
}

template <typename F> qsml_status_t by_dtype(int32_t dtype, F&& f) {
    return dtype == QSML_F32 ? f(static_cast<float*>(nullptr)) : f(static_cast<__half*>(nullptr));
}

// What the backward passes have in common: dz (or dg and du) into a workspace
// with the biases' gradients, then dx and the weights' gradients.
qsml_status_t backward(Context* ctx, const char* op, int32_t dtype, int32_t precision, int act, const Mat& x,
                       const Mat* w, int nw, const qsml_tdesc* dy, int64_t dy_ld, const qsml_tdesc* const* pre,
                       const qsml_tdesc* dx, const qsml_tdesc* const* dw, const qsml_tdesc* const* db) {
    const int64_t M = x.rows, K = x.cols, N = w[0].cols;
    const size_t es = dtype_size(dtype);
    bool want_dw = false, want_db = false;
    for (int i = 0; i < nw; ++i) {
        want_dw = want_dw || dw[i];
        want_db = want_db || db[i];
    }
    // How dz lies between its computation and the products.
    // binary32: in the three parts of the tensor cores, split once for both products; as
    // it is where the CUDA cores take it (FFMA, few rows).
    // binary16: rounding dz to 11 bits adds to dx and dw an error of the size of their own
    // rounding (1.4 times the error in all, however long the sums).  A dz of up to 2^16
    // elements is kept in two parts, 22 bits, which costs little there (256 x 256 x 256:
    // 16 us, in one part 13).  Beyond, it costs more than the bits are worth (512 x 1024 x
    // 1024: 20 us for 17; 16384 x 1024 x 2048: 271 for 157).
    // Without an activation dz = dy and needs no copy, binary32's split apart.
    // What binary16's dz lacks in range a power of two makes good (linear_grad.cu).
    const bool exact = act == QSML_ACT_NONE && nw == 1;
    const bool split = (dx || want_dw) && (dtype == QSML_F32 ? precision != QSML_MM_FP32_FFMA && M > 16
                                                             : !exact && M * N <= 65536);
    const bool plain = exact && !split;
    const size_t dz_bytes = !split ? es : dtype == QSML_F32 ? 6 : 4;  // an element
    Mat dz[2];
    Workspace ws(ctx);
    GradArgs g;
    g.M = M;
    g.N = N;
    g.act = act;
    g.dy = dy->data;
    g.dy_ld = dy_ld;
    g.pitch = line_pitch(N);
    g.plane = split ? g.pitch * M : 0;
    for (int i = 0; i < nw; ++i) {
        if (!plain) {
            if (act != QSML_ACT_NONE || nw == 2) g.pre[i] = pre[i]->data;
            if ((dx || want_dw) && M * N > 0) {
                // behind the first of binary16's: the scale of both
                const size_t bytes = static_cast<size_t>(M) * g.pitch * dz_bytes;
                const bool scaled = dtype == QSML_F16 && i == 0;
                QSML_TRY_STATUS(ws.get(bytes + (scaled ? sizeof(float) : 0), &g.dz[i]));
                if (scaled) g.unscale = reinterpret_cast<float*>(static_cast<char*>(g.dz[i]) + bytes);
                dz[i] = Mat{g.dz[i], M, N, g.pitch, 1, g.plane};
            }
        } else {
            dz[i] = Mat{dy->data, M, N, dy_ld, 1};
        }
        if (db[i]) {
            g.db[i].out = db[i]->data;
            g.db[i].out_dtype = db[i]->dtype;
        }
    }
    if (M == 0) {
        for (int i = 0; i < nw; ++i)
            if (db[i] && N)
                QSML_TRY_STATUS(check_cuda(ctx, cudaMemsetAsync(db[i]->data, 0, N * dtype_size(db[i]->dtype), ctx->stream), op));
    } else if (N > 0 && (want_db || (!plain && (dx || want_dw)))) {
        QSML_TRY_STATUS(by_dtype(dtype, [&](auto* t) { return run_grad<std::remove_pointer_t<decltype(t)>>(ctx, g, nw == 2); }));
    }
    Problem products[2];
    Problem* wanted[2];
    int n = 0;
    if (dx) {  // dz w^T, summed over the weights
        Problem& p = *(wanted[n] = &products[n]);
        ++n;
        p.M = M;
        p.N = K;
        p.K = N;
        p.segments = nw;
        for (int i = 0; i < nw; ++i) {
            p.a[i] = dz[i];
            p.b[i] = w[i].t();
        }
        p.e.y = dx->data;
        p.e.scale = g.unscale;
    }
    if (want_dw) {  // x^T dz
        Problem& p = *(wanted[n] = &products[n]);
        ++n;
        p.M = K;
        p.N = N;
        p.K = M;
        p.dual = nw == 2 && dw[0] && dw[1];
        p.e.scale = g.unscale;
        p.a[0] = x.t();
        if (p.dual) {
            p.b[0] = dz[0];
            p.b[1] = dz[1];
            p.e.pre[0] = dw[0]->data;
            p.e.pre[1] = dw[1]->data;
        } else {
            const int i = dw[0] ? 0 : 1;
            p.b[0] = dz[i];
            p.e.y = dw[i]->data;
        }
    }
    return run(ctx, dtype, precision, wanted, n);
}

}  // namespace
}  // namespace linear
}  // namespace qsml

using namespace qsml;
using namespace qsml::linear;

extern "C" qsml_status_t qsml_linear(qsml_ctx* handle, const qsml_tdesc* x, const qsml_tdesc* w, const qsml_tdesc* bias,
                                     int32_t act, const qsml_tdesc* residual, const qsml_tdesc* pre,
                                     const qsml_tdesc* y, int32_t precision) try {
    QSML_CTX(handle);
    const char* op = "qsml_linear";
    const Named all[6] = {{x, "x"}, {w, "w"}, {y, "y"}, {bias, "bias"}, {residual, "residual"}, {pre, "pre"}};
    QSML_TRY_STATUS(check_all(C_, all, 6, 3));
    QSML_TRY_STATUS(check_act(C_, op, act));
    QSML_TRY_STATUS(check_precision(C_, op, x->dtype, precision));
    Problem p;
    const char* wn[1] = {"w"};
    QSML_TRY_STATUS(check_xw(C_, op, x, &w, wn, 1, &p.a[0], &p.b[0]));
    p.M = p.a[0].rows;
    p.K = p.a[0].cols;
    p.N = p.b[0].cols;
    QSML_TRY_STATUS(check_vector(C_, op, Named{bias, "bias"}, x->dtype, p.N));
    QSML_TRY_STATUS(check_rows(C_, op, Named{y, "y"}, x, p.N));
    QSML_TRY_STATUS(check_rows(C_, op, Named{pre, "pre"}, x, p.N));
    QSML_TRY_STATUS(check_rows(C_, op, Named{residual, "residual"}, x, p.N, &p.e.res_ld));
    const Named in[4] = {{x, "x"}, {w, "w"}, {bias, "bias"}, {residual, "residual"}};
    const Named out[2] = {{y, "y"}, {pre, "pre"}};
    QSML_TRY_STATUS(check_overlap(C_, op, in, 4, out, 2, residual));
    p.e.bias[0] = bias ? bias->data : nullptr;
    p.e.bias_f32 = !bias || bias->dtype == QSML_F32;
    p.e.act = act;
    p.e.residual = residual ? residual->data : nullptr;
    p.e.pre[0] = pre ? pre->data : nullptr;
    p.e.y = y->data;
    return run(C_, x->dtype, precision, p);
} QSML_NO_THROW

extern "C" qsml_status_t qsml_linear_backward(qsml_ctx* handle, const qsml_tdesc* x, const qsml_tdesc* w, int32_t act,
                                              const qsml_tdesc* pre, const qsml_tdesc* dy, const qsml_tdesc* dx,
                                              const qsml_tdesc* dw, const qsml_tdesc* dbias, int32_t precision) try {
    QSML_CTX(handle);
    const char* op = "qsml_linear_backward";
    const Named all[7] = {{x, "x"}, {w, "w"}, {dy, "dy"}, {pre, "pre"}, {dx, "dx"}, {dw, "dw"}, {dbias, "dbias"}};
    QSML_TRY_STATUS(check_all(C_, all, 7, 3));
    QSML_TRY_STATUS(check_act(C_, op, act));
    QSML_TRY_STATUS(check_precision(C_, op, x->dtype, precision));
    if (act != QSML_ACT_NONE && !pre)
        return fail(C_, QSML_E_INVALID, op, "an activation's gradient needs pre, the product that the forward pass kept");
    Mat mx, mw;
    const char* wn[1] = {"w"};
    QSML_TRY_STATUS(check_xw(C_, op, x, &w, wn, 1, &mx, &mw));
    const int64_t K = mx.cols, N = mw.cols;
    int64_t dy_ld = 0;
    QSML_TRY_STATUS(check_rows(C_, op, Named{dy, "dy"}, x, N, &dy_ld));
    QSML_TRY_STATUS(check_rows(C_, op, Named{pre, "pre"}, x, N));
    QSML_TRY_STATUS(check_rows(C_, op, Named{dx, "dx"}, x, K));
    QSML_TRY_STATUS(check_dw(C_, op, Named{dw, "dw"}, x->dtype, K, N));
    QSML_TRY_STATUS(check_vector(C_, op, Named{dbias, "dbias"}, x->dtype, N));
    const Named in[4] = {{x, "x"}, {w, "w"}, {dy, "dy"}, {pre, "pre"}};
    const Named out[3] = {{dx, "dx"}, {dw, "dw"}, {dbias, "dbias"}};
    QSML_TRY_STATUS(check_overlap(C_, op, in, 4, out, 3, nullptr));
    return backward(C_, op, x->dtype, precision, act, mx, &mw, 1, dy, dy_ld, &pre, dx, &dw, &dbias);
} QSML_NO_THROW

extern "C" qsml_status_t qsml_gated_linear(qsml_ctx* handle, const qsml_tdesc* x, const qsml_tdesc* w_gate,
                                           const qsml_tdesc* w_up, const qsml_tdesc* b_gate, const qsml_tdesc* b_up,
                                           int32_t act, const qsml_tdesc* gate, const qsml_tdesc* up,
                                           const qsml_tdesc* y, int32_t precision) try {
    QSML_CTX(handle);
    const char* op = "qsml_gated_linear";
    const Named all[8] = {{x, "x"}, {w_gate, "w_gate"}, {w_up, "w_up"}, {y, "y"}, {b_gate, "b_gate"}, {b_up, "b_up"},
                          {gate, "gate"}, {up, "up"}};
    QSML_TRY_STATUS(check_all(C_, all, 8, 4));
    QSML_TRY_STATUS(check_act(C_, op, act));
    QSML_TRY_STATUS(check_precision(C_, op, x->dtype, precision));
    Problem p;
    p.dual = true;
    const qsml_tdesc* w[2] = {w_gate, w_up};
    const char* wn[2] = {"w_gate", "w_up"};
    QSML_TRY_STATUS(check_xw(C_, op, x, w, wn, 2, &p.a[0], p.b));
    p.M = p.a[0].rows;
    p.K = p.a[0].cols;
    p.N = p.b[0].cols;
    QSML_TRY_STATUS(check_vector(C_, op, Named{b_gate, "b_gate"}, x->dtype, p.N));
    QSML_TRY_STATUS(check_vector(C_, op, Named{b_up, "b_up"}, x->dtype, p.N));
    if (b_gate && b_up && b_gate->dtype != b_up->dtype)
        return fail(C_, QSML_E_DTYPE, op, "b_gate and b_up must have one dtype");
    QSML_TRY_STATUS(check_rows(C_, op, Named{y, "y"}, x, p.N));
    QSML_TRY_STATUS(check_rows(C_, op, Named{gate, "gate"}, x, p.N));
    QSML_TRY_STATUS(check_rows(C_, op, Named{up, "up"}, x, p.N));
    const Named in[5] = {{x, "x"}, {w_gate, "w_gate"}, {w_up, "w_up"}, {b_gate, "b_gate"}, {b_up, "b_up"}};
    const Named out[3] = {{y, "y"}, {gate, "gate"}, {up, "up"}};
    QSML_TRY_STATUS(check_overlap(C_, op, in, 5, out, 3, nullptr));
    p.e.bias[0] = b_gate ? b_gate->data : nullptr;
    p.e.bias[1] = b_up ? b_up->data : nullptr;
    p.e.bias_f32 = (!b_gate || b_gate->dtype == QSML_F32) && (!b_up || b_up->dtype == QSML_F32);
    p.e.act = act;
    p.e.pre[0] = gate ? gate->data : nullptr;
    p.e.pre[1] = up ? up->data : nullptr;
    p.e.y = y->data;
    return run(C_, x->dtype, precision, p);
} QSML_NO_THROW

extern "C" qsml_status_t qsml_gated_linear_backward(qsml_ctx* handle, const qsml_tdesc* x, const qsml_tdesc* w_gate,
                                                    const qsml_tdesc* w_up, int32_t act, const qsml_tdesc* gate,
                                                    const qsml_tdesc* up, const qsml_tdesc* dy, const qsml_tdesc* dx,
                                                    const qsml_tdesc* dw_gate, const qsml_tdesc* dw_up,
                                                    const qsml_tdesc* db_gate, const qsml_tdesc* db_up,
                                                    int32_t precision) try {
    QSML_CTX(handle);
    const char* op = "qsml_gated_linear_backward";
    const Named all[11] = {{x, "x"}, {w_gate, "w_gate"}, {w_up, "w_up"}, {gate, "gate"}, {up, "up"}, {dy, "dy"},
                           {dx, "dx"}, {dw_gate, "dw_gate"}, {dw_up, "dw_up"}, {db_gate, "db_gate"}, {db_up, "db_up"}};
    QSML_TRY_STATUS(check_all(C_, all, 11, 6));
    QSML_TRY_STATUS(check_act(C_, op, act));
    QSML_TRY_STATUS(check_precision(C_, op, x->dtype, precision));
    Mat mx, mw[2];
    const qsml_tdesc* w[2] = {w_gate, w_up};
    const char* wn[2] = {"w_gate", "w_up"};
    QSML_TRY_STATUS(check_xw(C_, op, x, w, wn, 2, &mx, mw));
    const int64_t K = mx.cols, N = mw[0].cols;
    int64_t dy_ld = 0;
    QSML_TRY_STATUS(check_rows(C_, op, Named{dy, "dy"}, x, N, &dy_ld));
    QSML_TRY_STATUS(check_rows(C_, op, Named{gate, "gate"}, x, N));
    QSML_TRY_STATUS(check_rows(C_, op, Named{up, "up"}, x, N));
    QSML_TRY_STATUS(check_rows(C_, op, Named{dx, "dx"}, x, K));
    QSML_TRY_STATUS(check_dw(C_, op, Named{dw_gate, "dw_gate"}, x->dtype, K, N));
    QSML_TRY_STATUS(check_dw(C_, op, Named{dw_up, "dw_up"}, x->dtype, K, N));
    QSML_TRY_STATUS(check_vector(C_, op, Named{db_gate, "db_gate"}, x->dtype, N));
    QSML_TRY_STATUS(check_vector(C_, op, Named{db_up, "db_up"}, x->dtype, N));
    const Named in[6] = {{x, "x"}, {w_gate, "w_gate"}, {w_up, "w_up"}, {gate, "gate"}, {up, "up"}, {dy, "dy"}};
    const Named out[5] = {{dx, "dx"}, {dw_gate, "dw_gate"}, {dw_up, "dw_up"}, {db_gate, "db_gate"}, {db_up, "db_up"}};
    QSML_TRY_STATUS(check_overlap(C_, op, in, 6, out, 5, nullptr));
    const qsml_tdesc* pre[2] = {gate, up};
    const qsml_tdesc* dw[2] = {dw_gate, dw_up};
    const qsml_tdesc* db[2] = {db_gate, db_up};
    return backward(C_, op, x->dtype, precision, act, mx, mw, 2, dy, dy_ld, pre, dx, dw, db);
} QSML_NO_THROW
