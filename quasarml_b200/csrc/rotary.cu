// Norms of queries and keys for each head with the rotation by positions, and the
// backward pass.  For a head's row x of D columns, with weight w (absent: no norm),
//   xh = x / sqrt(mean(x^2) + eps),  y = xh w,
// and of each rotated pair (a, b) of y, with the angle t = position * frequency,
//   (a cos t - b sin t,  b cos t + a sin t).
// The gradient g of y is the outputs' gradient turned back by t; then
//   dx = rstd (h - xh mean(h xh)),  h = g w,   dw = sum over tokens and heads of g xh.
// Bound by HBM: each element is read and written once (backward: two read, one written).
// A group of lanes holds a row, each lane 16 bytes of both halves of its pairs (or of
// neighbouring pairs), so a pair never leaves its lane and the row's sums are a few
// shuffles.  All heads of a token share its angles: the CTA computes them once, in binary64
// (at position 10^6 a binary32 angle is off by 0.03), reduced to a turn before the binary32
// sine and cosine.  The reference has neither.
#include "heads.cuh"

namespace qsml {
namespace {

using heads::from_f;
using heads::Pack;
using heads::to_f;
using heads::View;

constexpr int kThreads = 256;
constexpr int kMaxAxes = 4;
constexpr int kMaxD = 512;
constexpr int kMaxTokens = 8;  // of one pass of a CTA

struct RotaryArgs {
    View x[2], g[2], out[2];  // queries, keys; g: the outputs' gradients (backward)
    int H[2];
    const void* w[2];
    float* sums[2];  // partial sums [CTAs, D] of the weights' gradients
    const int* pos;
    int64_t pos_b, pos_s, pos_a;
    const float* freq;
    int ends[kMaxAxes];  // the pairs before ends[a] go by axis a or an earlier one
    int axes;
    int64_t T, S;  // tokens in all, and of one sequence
    int D, rot, pairs, w_f32;
    float eps;
};

template <typename T> __device__ __forceinline__ float weight(const void* w, int f32, int c) {
    return f32 ? static_cast<const float*>(w)[c] : to_f(static_cast<const T*>(w)[c]);
}

// (cos, sin) of pair i at token t.
__device__ __forceinline__ float2 turn(const RotaryArgs& a, int64_t b, int64_t s, int i) {
    int axis = 0;
    while (axis + 1 < a.axes && i >= a.ends[axis]) ++axis;
    const int64_t at = b * a.pos_b + s * a.pos_s + axis * a.pos_a;
    // position * frequency has 55 bits at most; a turn less whole turns, to 2^-22 at worst
    double u = static_cast<double>(a.pos[at]) * static_cast<double>(a.freq[i]) * 0.15915494309189533577;
    u -= rint(u);
    float sn, cs;
    sincospif(2.0f * static_cast<float>(u), &sn, &cs);
    return make_float2(cs, sn);
}

// A lane's chunk pair c of a row: where its two chunks of V columns start, the first pair it
// turns by, and whether it is turned.
template <int V> struct Chunk {
    int c0, c1, pair;
    bool turned;
    __device__ __forceinline__ Chunk(const RotaryArgs& a, int c) {
        const int half = a.rot / (2 * V);
        turned = c < half;
        if (V > 1 && a.pairs) {
            c0 = c * 2 * V;
            c1 = c0 + V;
            pair = c * V;
        } else if (V == 1 && a.pairs) {
            c0 = 2 * c;
            c1 = c0 + 1;
            pair = c;
        } else {
            c0 = turned ? c * V : a.rot + (c - half) * 2 * V;
            c1 = turned ? a.rot / 2 + c * V : c0 + V;
            pair = c * V;
        }
    }
};

// Turns a chunk pair by its V angles (sign -1: back).
template <int V> __device__ __forceinline__ void rotate(float (&p)[V], float (&q)[V], const float2 (&cs)[V], bool neighbours, float sign) {
    auto one = [&](float& a, float& b, float2 t) {
        const float s = sign * t.y, x = a, y = b;
        a = fmaf(x, t.x, -(y * s));
        b = fmaf(y, t.x, x * s);
    };
    if (V > 1 && neighbours) {
#pragma unroll
        for (int e = 0; e + 1 < V; e += 2) {
            one(p[e], p[e + 1], cs[e / 2]);
            one(q[e], q[e + 1], cs[V / 2 + e / 2]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) one(p[e], q[e], cs[e]);
    }
}

template <typename T, int V> __device__ __forceinline__ void load(float (&r)[V], const T* p) {
    const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
    for (int e = 0; e < V; ++e) r[e] = to_f(v.v[e]);
}
template <typename T, int V> __device__ __forceinline__ void store(const float (&r)[V], T* p) {
    Pack<T, V> v;
#pragma unroll
    for (int e = 0; e < V; ++e) from_f(r[e], v.v[e]);
    *reinterpret_cast<Pack<T, V>*>(p) = v;
}

// Row r of a token: head r of the queries, or r - H[0] of the keys.
__device__ __forceinline__ int64_t row_at(const View& v, int64_t b, int64_t s, int h) { return b * v.b + s * v.s + h * v.h; }

// NC chunk pairs of V columns a lane; `lanes` (a power of two) lanes a row; `tokens` tokens a
// pass of the CTA.
template <typename T, int V, int NC, bool BWD>
__global__ void __launch_bounds__(kThreads) k_norm_rotary(const __grid_constant__ RotaryArgs a, int lanes, int tokens) {
    __shared__ float2 angle[kMaxTokens * kMaxD / 2];
    pdl_begin();
    const int lane = threadIdx.x & (lanes - 1), slot = threadIdx.x / lanes;
    const int slots = kThreads / lanes / tokens;  // rows of one token in flight
    const int sub = slot / slots, row0 = slot % slots;
    const int pairs = a.rot / 2, rows = a.H[0] + a.H[1], chunks = a.D / (2 * V);
    const float inv_d = 1.0f / static_cast<float>(a.D);
    float dw[2][BWD ? NC : 1][BWD ? 2 * V : 1] = {};
    for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * tokens; t0 < a.T; t0 += static_cast<int64_t>(gridDim.x) * tokens) {
        const int64_t t = t0 + sub;
        const bool here = t < a.T;
        const int64_t b = here ? t / a.S : 0, s = here ? t - b * a.S : 0;
        for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
            const int64_t ti = t0 + i / pairs;
            if (ti < a.T) angle[i] = turn(a, ti / a.S, ti % a.S, i % pairs);
        }
        __syncthreads();
        float2 cs[NC][V];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const Chunk<V> c(a, lane + n * lanes);
#pragma unroll
            for (int e = 0; e < V; ++e) cs[n][e] = c.turned && here ? angle[sub * pairs + c.pair + e] : make_float2(1.0f, 0.0f);
        }
        // the group's lanes stay together: every lane of a warp goes through as many rows
        for (int r = row0; r - row0 < rows; r += slots) {
            const int which = r < a.H[0] ? 0 : 1;
            const bool live = here && r < rows;
            const int h = which ? r - a.H[0] : r;
            const void* w = a.w[which];
            const T* x = reinterpret_cast<const T*>(a.x[which].p) + (live ? row_at(a.x[which], b, s, h) : 0);
            float p[NC][2][V], sq = 0.0f;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                const Chunk<V> c(a, lane + n * lanes);
#pragma unroll
                for (int e = 0; e < V; ++e) p[n][0][e] = p[n][1][e] = 0.0f;
                if (live && lane + n * lanes < chunks) {
                    load<T, V>(p[n][0], x + c.c0);
                    load<T, V>(p[n][1], x + c.c1);
                }
#pragma unroll
                for (int e = 0; e < V; ++e) sq = fmaf(p[n][0][e], p[n][0][e], fmaf(p[n][1][e], p[n][1][e], sq));
            }
            float g[BWD ? NC : 1][2][V];
            float hx = 0.0f;
            if constexpr (BWD) {
                const T* y = reinterpret_cast<const T*>(a.g[which].p) + (live ? row_at(a.g[which], b, s, h) : 0);
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    const Chunk<V> c(a, lane + n * lanes);
#pragma unroll
                    for (int e = 0; e < V; ++e) g[n][0][e] = g[n][1][e] = 0.0f;
                    if (live && lane + n * lanes < chunks) {
                        load<T, V>(g[n][0], y + c.c0);
                        load<T, V>(g[n][1], y + c.c1);
                        if (c.turned) rotate<V>(g[n][0], g[n][1], cs[n], a.pairs, -1.0f);
                        if (w) {
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int e = 0; e < V; ++e)
                                    hx = fmaf(g[n][i][e] * weight<T>(w, a.w_f32, (i ? c.c1 : c.c0) + e), p[n][i][e], hx);
                        }
                    }
                }
            }
            for (int m = lanes >> 1; m >= 1; m >>= 1) {
                sq += __shfl_xor_sync(0xffffffffu, sq, m);
                if (BWD) hx += __shfl_xor_sync(0xffffffffu, hx, m);
            }
            const float rstd = w ? 1.0f / sqrtf(fmaf(sq, inv_d, a.eps)) : 1.0f;
            if (!live) continue;
            T* out = a.out[which].p ? reinterpret_cast<T*>(a.out[which].p) + row_at(a.out[which], b, s, h) : nullptr;
            const float along = hx * rstd * rstd * inv_d;  // mean(h xh) rstd, that x takes
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                if (lane + n * lanes >= chunks) continue;
                const Chunk<V> c(a, lane + n * lanes);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const int col = (i ? c.c1 : c.c0) + e;
                        if constexpr (BWD) {
                            if (w) {
                                const float xv = p[n][i][e];
                                if (which == 0)
                                    dw[0][n][i * V + e] = fmaf(g[n][i][e], xv * rstd, dw[0][n][i * V + e]);
                                else
                                    dw[1][n][i * V + e] = fmaf(g[n][i][e], xv * rstd, dw[1][n][i * V + e]);
                                g[n][i][e] = rstd * fmaf(-xv, along, g[n][i][e] * weight<T>(w, a.w_f32, col));
                            }
                        } else if (w) {
                            p[n][i][e] = p[n][i][e] * rstd * weight<T>(w, a.w_f32, col);
                        }
                    }
                if constexpr (BWD) {
                    if (out) {
                        store<T, V>(g[n][0], out + c.c0);
                        store<T, V>(g[n][1], out + c.c1);
                    }
                } else {
                    if (c.turned) rotate<V>(p[n][0], p[n][1], cs[n], a.pairs, 1.0f);
                    store<T, V>(p[n][0], out + c.c0);
                    store<T, V>(p[n][1], out + c.c1);
                }
            }
        }
        __syncthreads();
    }
    if constexpr (BWD) {
        // the CTA's rows joined in the order of their slots
        __shared__ float part[kThreads * 2 * V * NC];  // [slots of the CTA][D at most]
        const int all = kThreads / lanes;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (!a.sums[k]) continue;
            __syncthreads();
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                if (lane + n * lanes >= chunks) continue;
                const Chunk<V> c(a, lane + n * lanes);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    part[slot * a.D + c.c0 + e] = dw[k][n][e];
                    part[slot * a.D + c.c1 + e] = dw[k][n][V + e];
                }
            }
            __syncthreads();
            for (int c = threadIdx.x; c < a.D; c += kThreads) {
                float v = 0.0f;
                for (int i = 0; i < all; ++i) v += part[i * a.D + c];
                a.sums[k][static_cast<int64_t>(blockIdx.x) * a.D + c] = v;
            }
        }
    }
}

template <typename T, bool BWD> qsml_status_t launch(Context* ctx, const RotaryArgs& a, int vec, unsigned grid, int lanes, int tokens) {
    cudaError_t e = cudaSuccess;
    const int chunks = a.D / (2 * vec);
    const bool one = chunks <= 32;
    auto go = [&](auto kernel) { e = launch_pdl(kernel, dim3(grid), dim3(kThreads), 0, ctx->stream, a, lanes, tokens); };
    constexpr int FULL = 16 / sizeof(T);
    if (vec == FULL) {
        if constexpr (sizeof(T) == 2)
            go(k_norm_rotary<T, FULL, 1, BWD>);
        else
            one ? go(k_norm_rotary<T, FULL, 1, BWD>) : go(k_norm_rotary<T, FULL, 2, BWD>);
    } else if (vec == 2) {
        one ? go(k_norm_rotary<T, 2, 1, BWD>) : go(k_norm_rotary<T, 2, 4, BWD>);
    } else {
        one ? go(k_norm_rotary<T, 1, 1, BWD>) : go(k_norm_rotary<T, 1, 8, BWD>);
    }
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_norm_rotary");
    return after_launch(ctx, BWD ? "k_norm_rotary_bwd" : "k_norm_rotary");
}

// The checks that both directions share; fills what the kernel takes but for gradients and outputs.
struct Inputs {
    const qsml_tdesc *q, *k, *wq, *wk, *pos, *freq;
    float eps;
    const int32_t* sections;
    int32_t n_sections, pairing;
};

qsml_status_t check_inputs(Context* ctx, const char* op, const Inputs& in, RotaryArgs* a, heads::Dims* dq, heads::Dims* dk) {
    using heads::fail;
    const qsml_tdesc *q = in.q, *k = in.k;
    const qsml_tdesc* all[6] = {q, in.pos, in.freq, k, in.wq, in.wk};
    const char* names[6] = {"q", "positions", "frequencies", "k", "wq", "wk"};
    for (int i = 0; i < 6; ++i)
        if (i < 3 || all[i]) QSML_TRY_STATUS(check_desc(ctx, all[i], names[i]));
    if (q->dtype != QSML_F32 && q->dtype != QSML_F16) return fail(ctx, QSML_E_DTYPE, op, "q must be F32 or F16");
    if (in.pairing != QSML_ROTARY_HALVES && in.pairing != QSML_ROTARY_PAIRS) return fail(ctx, QSML_E_INVALID, op, "unknown pairing");
    if (!(in.eps >= 0.0f && in.eps < INFINITY)) return fail(ctx, QSML_E_INVALID, op, "eps must be finite and not negative");
    QSML_TRY_STATUS((heads::view_of(ctx, op, {q, "q"}, false, dq, &a->x[0])));
    *dk = heads::Dims{dq->B, dq->S, 0, dq->D};
    if (k) {
        if (k->dtype != q->dtype) return fail(ctx, QSML_E_DTYPE, op, "k must have q's dtype");
        if (k->ndim != q->ndim) return fail(ctx, QSML_E_SHAPE, op, "q and k must have one rank");
        QSML_TRY_STATUS((heads::view_of(ctx, op, {k, "k"}, false, dk, &a->x[1])));
        if (dk->B != dq->B || dk->S != dq->S || dk->D != dq->D)
            return fail(ctx, QSML_E_SHAPE, op, "q and k must have the same tokens and columns");
    }
    if (dq->D % 2) return fail(ctx, QSML_E_SHAPE, op, "the heads need an even number of columns");
    if (dq->D > kMaxD) return fail(ctx, QSML_E_UNSUPPORTED, op, "heads of more than 512 columns");
    if (dq->H + dk->H > INT32_MAX / 2) return fail(ctx, QSML_E_UNSUPPORTED, op, "too many heads");
    if (!k && in.wk) return fail(ctx, QSML_E_INVALID, op, "wk without k");
    const qsml_tdesc* w[2] = {in.wq, in.wk};
    a->w_f32 = 1;
    for (int i = 0; i < 2; ++i) {
        a->w[i] = w[i] ? w[i]->data : nullptr;
        if (!w[i]) continue;
        if (w[i]->dtype != QSML_F32 && w[i]->dtype != q->dtype)
            return fail(ctx, QSML_E_DTYPE, op, std::string(names[4 + i]) + " must be F32 or q's dtype");
        if (w[i]->ndim != 1 || w[i]->shape[0] != dq->D)
            return fail(ctx, QSML_E_SHAPE, op, std::string(names[4 + i]) + " must be [columns]");
        if (!is_contiguous(w[i])) return fail(ctx, QSML_E_UNSUPPORTED, op, std::string(names[4 + i]) + " must be contiguous");
        a->w_f32 = w[i]->dtype == QSML_F32;
    }
    if (in.wq && in.wk && in.wq->dtype != in.wk->dtype) return fail(ctx, QSML_E_DTYPE, op, "wq and wk must have one dtype");
    if (in.freq->dtype != QSML_F32) return fail(ctx, QSML_E_DTYPE, op, "frequencies must be F32");
    if (in.freq->ndim != 1 || in.freq->shape[0] < 1 || 2 * in.freq->shape[0] > dq->D)
        return fail(ctx, QSML_E_SHAPE, op, "frequencies must be [pairs], between one and half the columns");
    if (!is_contiguous(in.freq)) return fail(ctx, QSML_E_UNSUPPORTED, op, "frequencies must be contiguous");
    const int64_t pairs = in.freq->shape[0];
    if (in.pos->dtype != QSML_I32) return fail(ctx, QSML_E_DTYPE, op, "positions must be I32");
    if (in.n_sections < 0 || in.n_sections > kMaxAxes || (in.n_sections > 0 && !in.sections))
        return fail(ctx, QSML_E_INVALID, op, "sections: up to four counts of pairs");
    int64_t end = 0;
    a->axes = in.n_sections > 0 ? in.n_sections : 1;
    for (int i = 0; i < in.n_sections; ++i) {
        if (in.sections[i] < 0) return fail(ctx, QSML_E_INVALID, op, "a section has a negative count");
        end += in.sections[i];
        a->ends[i] = static_cast<int>(end < pairs ? end : pairs);
    }
    if (in.n_sections > 0 && end != pairs) return fail(ctx, QSML_E_SHAPE, op, "the sections must add up to the number of frequencies");
    // positions [tokens] ([sequences, tokens]), with a last dim of axes where there are sections
    const int lead = q->ndim - 2, want = lead + (in.n_sections > 0 ? 1 : 0);
    bool ok = in.pos->ndim == want;
    for (int i = 0; ok && i < lead; ++i) ok = in.pos->shape[i] == q->shape[i];
    if (ok && want > lead) ok = in.pos->shape[lead] == in.n_sections;
    if (!ok) return fail(ctx, QSML_E_SHAPE, op, "positions must be [tokens] (as q has them), and one for each section");
    a->pos = static_cast<const int*>(in.pos->data);
    a->pos_b = lead == 2 ? in.pos->stride[0] : 0;
    a->pos_s = in.pos->stride[lead - 1];
    a->pos_a = want > lead ? in.pos->stride[lead] : 0;
    a->freq = static_cast<const float*>(in.freq->data);
    a->H[0] = static_cast<int>(dq->H);
    a->H[1] = static_cast<int>(dk->H);
    a->S = dq->S;
    a->T = dq->B * dq->S;
    a->D = static_cast<int>(dq->D);
    a->rot = static_cast<int>(2 * pairs);
    a->pairs = in.pairing == QSML_ROTARY_PAIRS;
    a->eps = in.eps;
    return QSML_OK;
}

// One of the outputs, shaped as `like`.
qsml_status_t check_output(Context* ctx, const char* op, heads::Named t, const qsml_tdesc* like, bool output, View* v) {
    if (!t.d) return QSML_OK;
    if (t.d->dtype != like->dtype) return heads::fail(ctx, QSML_E_DTYPE, op, std::string(t.name) + " must have q's dtype");
    bool ok = t.d->ndim == like->ndim;
    for (int i = 0; ok && i < like->ndim; ++i) ok = t.d->shape[i] == like->shape[i];
    if (!ok) return heads::fail(ctx, QSML_E_SHAPE, op, std::string(t.name) + " has the wrong shape");
    heads::Dims d;
    return heads::view_of(ctx, op, t, output, &d, v);
}

// The widest chunks that sizes and alignment of all rows allow: 16 bytes, two columns, one.
int chunk_of(const RotaryArgs& a, int es, bool backward) {
    for (int v : {16 / es, 2}) {
        bool ok = a.D % (2 * v) == 0 && a.rot % (2 * v) == 0;
        for (int i = 0; i < 2; ++i) {
            if (!a.H[i]) continue;
            ok = ok && heads::rows_on(a.x[i], es, v * es);
            if (a.out[i].p) ok = ok && heads::rows_on(a.out[i], es, v * es);
            if (backward) ok = ok && heads::rows_on(a.g[i], es, v * es);
        }
        if (ok) return v;
    }
    return 1;
}

// Lanes a row (a power of two), and tokens a pass: as many as keep every lane at a row.
void shape_of(const RotaryArgs& a, int vec, int* lanes, int* tokens) {
    const int chunks = a.D / (2 * vec);
    *lanes = 1;
    while (*lanes < chunks && *lanes < 32) *lanes *= 2;
    *tokens = 1;
    while (*tokens < kMaxTokens && kThreads / *lanes / (*tokens * 2) >= a.H[0] + a.H[1]) *tokens *= 2;
}

}  // namespace
}  // namespace qsml

using namespace qsml;

extern "C" qsml_status_t qsml_norm_rotary(qsml_ctx* handle, const qsml_tdesc* q, const qsml_tdesc* k, const qsml_tdesc* wq,
                                          const qsml_tdesc* wk, float eps, const qsml_tdesc* positions,
                                          const qsml_tdesc* frequencies, const int32_t* sections, int32_t n_sections,
                                          int32_t pairing, const qsml_tdesc* q_out, const qsml_tdesc* k_out) try {
    QSML_CTX(handle);
    const char* op = "qsml_norm_rotary";
    RotaryArgs a = {};
    heads::Dims dq, dk;
    const Inputs inputs{q, k, wq, wk, positions, frequencies, eps, sections, n_sections, pairing};
    QSML_TRY_STATUS(check_inputs(C_, op, inputs, &a, &dq, &dk));
    if ((k == nullptr) != (k_out == nullptr)) return heads::fail(C_, QSML_E_INVALID, op, "k and k_out go together");
    QSML_TRY_STATUS(check_desc(C_, q_out, "q_out"));
    if (k_out) QSML_TRY_STATUS(check_desc(C_, k_out, "k_out"));
    QSML_TRY_STATUS((check_output(C_, op, {q_out, "q_out"}, q, true, &a.out[0])));
    QSML_TRY_STATUS((check_output(C_, op, {k_out, "k_out"}, k, true, &a.out[1])));
    const heads::Named in[6] = {{q, "q"}, {k, "k"}, {wq, "wq"}, {wk, "wk"}, {positions, "positions"}, {frequencies, "frequencies"}};
    const heads::Named out[2] = {{q_out, "q_out"}, {k_out, "k_out"}};
    QSML_TRY_STATUS(heads::check_overlap(C_, op, in, 6, out, 2, 2));
    if (a.T == 0 || a.D == 0 || a.H[0] + a.H[1] == 0) return QSML_OK;
    const int es = dtype_size(q->dtype), vec = chunk_of(a, es, false);
    int lanes, tokens;
    shape_of(a, vec, &lanes, &tokens);
    const int64_t passes = (a.T + tokens - 1) / tokens;
    const unsigned grid = static_cast<unsigned>(passes < 1 << 20 ? passes : 1 << 20);
    return q->dtype == QSML_F16 ? launch<__half, false>(C_, a, vec, grid, lanes, tokens)
                                : launch<float, false>(C_, a, vec, grid, lanes, tokens);
} QSML_NO_THROW

extern "C" qsml_status_t qsml_norm_rotary_backward(qsml_ctx* handle, const qsml_tdesc* q, const qsml_tdesc* k,
                                                   const qsml_tdesc* wq, const qsml_tdesc* wk, float eps,
                                                   const qsml_tdesc* positions, const qsml_tdesc* frequencies,
                                                   const int32_t* sections, int32_t n_sections, int32_t pairing,
                                                   const qsml_tdesc* dq_out, const qsml_tdesc* dk_out, const qsml_tdesc* dq,
                                                   const qsml_tdesc* dk, const qsml_tdesc* dwq, const qsml_tdesc* dwk) try {
    QSML_CTX(handle);
    const char* op = "qsml_norm_rotary_backward";
    RotaryArgs a = {};
    heads::Dims nq, nk;
    const Inputs inputs{q, k, wq, wk, positions, frequencies, eps, sections, n_sections, pairing};
    QSML_TRY_STATUS(check_inputs(C_, op, inputs, &a, &nq, &nk));
    if ((k == nullptr) != (dk_out == nullptr)) return heads::fail(C_, QSML_E_INVALID, op, "k and dk_out go together");
    if (!k && dk) return heads::fail(C_, QSML_E_INVALID, op, "dk without k");
    if ((dwq && !wq) || (dwk && !wk)) return heads::fail(C_, QSML_E_INVALID, op, "the gradient of an absent weight");
    const heads::Named out[4] = {{dq, "dq"}, {dk, "dk"}, {dwq, "dwq"}, {dwk, "dwk"}};
    QSML_TRY_STATUS(check_desc(C_, dq_out, "dq_out"));
    if (dk_out) QSML_TRY_STATUS(check_desc(C_, dk_out, "dk_out"));
    for (const auto& t : out)
        if (t.d) QSML_TRY_STATUS(check_desc(C_, t.d, t.name));
    QSML_TRY_STATUS((check_output(C_, op, {dq_out, "dq_out"}, q, false, &a.g[0])));
    QSML_TRY_STATUS((check_output(C_, op, {dk_out, "dk_out"}, k, false, &a.g[1])));
    QSML_TRY_STATUS((check_output(C_, op, {dq, "dq"}, q, true, &a.out[0])));
    QSML_TRY_STATUS((check_output(C_, op, {dk, "dk"}, k, true, &a.out[1])));
    for (int i = 2; i < 4; ++i) {
        const qsml_tdesc* d = out[i].d;
        if (!d) continue;
        if (d->dtype != QSML_F32 && d->dtype != q->dtype)
            return heads::fail(C_, QSML_E_DTYPE, op, std::string(out[i].name) + " must be F32 or q's dtype");
        if (d->ndim != 1 || d->shape[0] != nq.D) return heads::fail(C_, QSML_E_SHAPE, op, std::string(out[i].name) + " must be [columns]");
        if (!is_contiguous(d)) return heads::fail(C_, QSML_E_UNSUPPORTED, op, std::string(out[i].name) + " must be contiguous");
    }
    // the gradients may take the place of the outputs' gradients
    const heads::Named in[8] = {{dq_out, "dq_out"}, {dk_out, "dk_out"}, {q, "q"}, {k, "k"}, {wq, "wq"}, {wk, "wk"},
                                {positions, "positions"}, {frequencies, "frequencies"}};
    QSML_TRY_STATUS(heads::check_overlap(C_, op, in, 8, out, 4, 2));
    if (a.D == 0 || (!dq && !dk && !dwq && !dwk)) return QSML_OK;
    // with no rows a weight's gradient is 0
    const qsml_tdesc* dw[2] = {dwq, dwk};
    for (int i = 0; i < 2; ++i)
        if (dw[i] && (a.T == 0 || a.H[i] == 0))
            QSML_TRY_STATUS(check_cuda(C_, cudaMemsetAsync(dw[i]->data, 0, a.D * dtype_size(dw[i]->dtype), C_->stream), op));
    if (a.T == 0) return QSML_OK;
    // heads whose gradients nobody wants are left out
    if (!dq && !dwq) a.H[0] = 0;
    if (!dk && !dwk) a.H[1] = 0;
    if (a.H[0] + a.H[1] == 0) return QSML_OK;
    const int es = dtype_size(q->dtype), vec = chunk_of(a, es, true);
    int lanes, tokens;
    shape_of(a, vec, &lanes, &tokens);
    const int64_t passes = (a.T + tokens - 1) / tokens;
    const int64_t most = 4 * static_cast<int64_t>(C_->num_sms);
    const unsigned grid = static_cast<unsigned>(passes < most ? passes : most);
    Workspace ws(C_);
    ColumnSum sums[2];
    for (int i = 0; i < 2; ++i) {
        if (!dw[i] || !a.H[i]) continue;
        void* p = nullptr;
        QSML_TRY_STATUS(ws.get(sizeof(float) * a.D * grid, &p));
        a.sums[i] = static_cast<float*>(p);
        sums[i] = ColumnSum{a.sums[i], dw[i]->data, dw[i]->dtype};
    }
    QSML_TRY_STATUS((q->dtype == QSML_F16 ? launch<__half, true>(C_, a, vec, grid, lanes, tokens)
                                          : launch<float, true>(C_, a, vec, grid, lanes, tokens)));
    return finish_column_sums(C_, sums[0], sums[1], grid, a.D);
} QSML_NO_THROW
