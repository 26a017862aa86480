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
// shuffles.  A CTA has lanes for all heads of a token and goes from token to token, so that a
// lane keeps its columns of the weight (and sums their gradient) in registers; the next row is
// loaded, and the next token's angles are computed, under the present one.  Angles are shared by
// the heads and taken in binary64 (at position 10^6 a binary32 angle is off by 0.03), less whole
// turns, before the binary32 sine and cosine.  The reference has neither.
#include <algorithm>
#include <type_traits>

#include "heads.cuh"
#include "packed.cuh"

namespace qsml {
namespace {

using heads::from_f;
using heads::Pack;
using heads::to_f;
using heads::View;

// Threads of a CTA, at most, and CTAs a SM that registers are to be had for.  Forward: 80 registers, 81 us
// of 16384 tokens of 40 heads of 128 in binary16 (4 x 192 threads 80, 5 x 160 82, 6 x 160 90, and 109 with two
// rows on their way instead of one).  Backward: 128, for these heads without spills, 122 us (2 x 320 threads 154,
// 4 x 128 131); the kernels of wide heads (binary32 beyond 256 columns, and those that no vector fits beyond 128)
// spill 96 to 204 bytes.
constexpr int most_threads(bool backward) { return backward ? 160 : 384; }
constexpr int least_ctas(bool backward) { return backward ? 3 : 2; }
constexpr int kMaxAxes = 4;
constexpr int kMaxD = 512;

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
    int T, S;  // tokens in all, and of one sequence
    int D, rot, pairs, w_f32;
    float eps;
};

// Sequence and place of token t.
struct Token {
    int b, s;
    __device__ __forceinline__ Token(const RotaryArgs& a, int t) {
        b = t < a.S ? 0 : static_cast<int>(static_cast<unsigned>(t) / static_cast<unsigned>(a.S));
        s = t - b * a.S;
    }
};

// (cos, sin) of pair i of a token.
__device__ __forceinline__ float2 turn(const RotaryArgs& a, int b, int s, int i) {
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
template <int V, bool PAIRS> struct Chunk {
    int c0, c1, pair;
    bool turned;
    __device__ __forceinline__ Chunk(const RotaryArgs& a, int c) {
        const int half = a.rot / (2 * V);
        turned = c < half;
        c0 = PAIRS || !turned ? (PAIRS ? c * 2 * V : a.rot + (c - half) * 2 * V) : c * V;
        c1 = PAIRS || !turned ? c0 + V : a.rot / 2 + c * V;
        pair = c * V;
    }
};

// Arithmetic on V columns: packed pairs, or one number.
__device__ __forceinline__ float mul2(float a, float b) { return a * b; }
__device__ __forceinline__ float fma2(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float sum2(float a) { return a; }
template <int V> struct Cols {
    using E = typename std::conditional<V == 1, float, P2>::type;
    static constexpr int N = V == 1 ? 1 : V / 2;
    E v[N];
    static __device__ __forceinline__ E all(float a) {
        if constexpr (V == 1)
            return a;
        else
            return both(a);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (E& x : v) x = all(0.0f);
    }
    template <typename T> __device__ __forceinline__ void from(const Pack<T, V>& p) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if constexpr (V == 1) {
                v[i] = to_f(p.v[i]);
            } else if constexpr (sizeof(T) == 2) {
                const float2 f = __half22float2(reinterpret_cast<const __half2*>(&p)[i]);
                v[i] = pack(f.x, f.y);
            } else
                v[i] = pack(to_f(p.v[2 * i]), to_f(p.v[2 * i + 1]));
    }
    template <typename T> __device__ __forceinline__ void store(T* to) const {
        Pack<T, V> p;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if constexpr (V == 1) {
                from_f(v[i], p.v[i]);
            } else {
                const float2 f = unpack(v[i]);
                if constexpr (sizeof(T) == 2) {
                    reinterpret_cast<__half2*>(&p)[i] = __floats2half2_rn(f.x, f.y);
                } else {
                    p.v[2 * i] = f.x;
                    p.v[2 * i + 1] = f.y;
                }
            }
        *reinterpret_cast<Pack<T, V>*>(to) = p;
    }
};

// Turns a chunk pair by V angles, their cosines and sines (BACK: by their opposites).
template <int V, bool PAIRS, bool BACK>
__device__ __forceinline__ void rotate(Cols<V>& p, Cols<V>& q, const float* cosine, const float* sine) {
    const Pack<float, V> c = *reinterpret_cast<const Pack<float, V>*>(cosine), s = *reinterpret_cast<const Pack<float, V>*>(sine);
    if constexpr (V > 1 && PAIRS) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            P2& x = e < V / 2 ? p.v[e] : q.v[e - V / 2];
            const float2 f = unpack(x);
            const float t = BACK ? -s.v[e] : s.v[e];
            x = fma2(pack(f.y, f.x), pack(-t, t), mul2(x, both(c.v[e])));
        }
    } else {
        Cols<V> cc, ss, ns;
        cc.from(c);
#pragma unroll
        for (int i = 0; i < Cols<V>::N; ++i) {
            if constexpr (V == 1) {
                ss.v[i] = s.v[i];
                ns.v[i] = -s.v[i];
            } else {
                ss.v[i] = pack(s.v[2 * i], s.v[2 * i + 1]);
                ns.v[i] = pack(-s.v[2 * i], -s.v[2 * i + 1]);
            }
            const auto x = p.v[i], y = q.v[i];
            p.v[i] = fma2(y, BACK ? ss.v[i] : ns.v[i], mul2(x, cc.v[i]));
            q.v[i] = fma2(x, BACK ? ns.v[i] : ss.v[i], mul2(y, cc.v[i]));
        }
    }
}

// How a CTA's lanes are laid over a token's rows: groups of `lanes` (a power of two), the first
// slots[0] of them for queries, the next slots[1] for keys, each for `rounds` rows; tokens in batches, whose angles are computed together.
struct Shape {
    int vec, lanes, slots[2], rounds, threads, batch;
    size_t smem;
};

// NC chunk pairs of V columns a lane.
template <typename T, int V, int NC, bool PAIRS, bool BWD>
__global__ void __launch_bounds__(most_threads(BWD), least_ctas(BWD)) k_norm_rotary(const __grid_constant__ RotaryArgs a, Shape sh) {
    extern __shared__ float4 shared[];  // cosines and sines [2][batch][2][pairs]; backward: then [slots][D] partial sums
    float* angle = reinterpret_cast<float*>(shared);
    pdl_begin();
    const int lane = threadIdx.x & (sh.lanes - 1), slot = threadIdx.x / sh.lanes;
    const int which = slot < sh.slots[0] ? 0 : 1, row0 = which ? slot - sh.slots[0] : slot, step = sh.slots[which];
    const int rows = which && row0 >= step ? 0 : a.H[which];  // lanes that fill the last warp have none
    const int pairs = a.rot / 2, chunks = a.D / (2 * V);
    const float inv_d = 1.0f / static_cast<float>(a.D);
    const bool normed = a.w[which] != nullptr;
    using Chunks = Chunk<V, PAIRS>;
    constexpr int N = Cols<V>::N;
    Cols<V> wt[NC][2], dw[BWD ? NC : 1][2];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const Chunks c(a, lane + n * sh.lanes);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if constexpr (BWD) dw[n][k].zero();
            Pack<float, V> w;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int col = (k ? c.c1 : c.c0) + e;
                w.v[e] = 1.0f;
                if (normed && lane + n * sh.lanes < chunks)
                    w.v[e] = a.w_f32 ? static_cast<const float*>(a.w[which])[col] : to_f(static_cast<const T*>(a.w[which])[col]);
            }
            wt[n][k].from(w);
        }
    }
    // a lane's rows of the CTA's tokens come one after the other
    Pack<T, V> nx[NC][2], ng[BWD ? NC : 1][2];
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                from_f(0.0f, nx[n][k].v[e]);  // what no row is read into stays 0
                if constexpr (BWD) from_f(0.0f, ng[n][k].v[e]);
            }
    // the lane's first row of token 0 and the step to the next token; sequences and further rounds, which
    // are rare, by the arguments
    struct Base {
        T* p;
        int64_t s;
        __device__ __forceinline__ Base(const View& v, int row) : p(reinterpret_cast<T*>(v.p) + row * v.h), s(v.s) {}
        __device__ __forceinline__ T* at(const View& v, const Token& k, int more) const {
            T* q = p + k.s * s;
            if (k.b) q += k.b * v.b;
            if (more) q += more * v.h;
            return q;
        }
    };
    const Base bx(a.x[which], row0), bg(a.g[which], row0), bo(a.out[which], row0);
    const bool wanted = a.out[which].p != nullptr;
    auto fetch = [&](int t, int r) {
        if (t >= a.T || r >= rows) return;
        const Token k(a, t);
        const T* x = bx.at(a.x[which], k, r - row0);
        const T* g = BWD ? bg.at(a.g[which], k, r - row0) : nullptr;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            if (lane + n * sh.lanes >= chunks) continue;
            const Chunks c(a, lane + n * sh.lanes);
            nx[n][0] = *reinterpret_cast<const Pack<T, V>*>(x + c.c0);
            nx[n][1] = *reinterpret_cast<const Pack<T, V>*>(x + c.c1);
            if constexpr (BWD) {
                ng[n][0] = *reinterpret_cast<const Pack<T, V>*>(g + c.c0);
                ng[n][1] = *reinterpret_cast<const Pack<T, V>*>(g + c.c1);
            }
        }
    };
    auto angles = [&](int t0, float* to) {
        for (int i = threadIdx.x; i < sh.batch * pairs; i += blockDim.x) {
            const int j = i / pairs;
            if (j < a.T - t0) {
                const Token k(a, t0 + j);
                const float2 cs = turn(a, k.b, k.s, i - j * pairs);
                to[i + j * pairs] = cs.x;
                to[i + (j + 1) * pairs] = cs.y;
            }
        }
    };
    const int64_t stride = static_cast<int64_t>(gridDim.x) * sh.batch;
    int t = blockIdx.x * sh.batch;
    fetch(t, row0);
    angles(t, angle);
    int buffer = 0, at = 0;  // of the angles; in the batch
    while (t < a.T) {
        if (at == 0) __syncthreads();
        const bool more = at + 1 < sh.batch && t + 1 < a.T;
        const int first = t - at, then = stride < a.T - first ? first + static_cast<int>(stride) : a.T;
        const int after = more ? t + 1 : then;
        const Token tk(a, t);
        const float* cs_at = angle + 2 * (buffer * sh.batch + at) * pairs;
        // every lane of a warp goes through as many rows
        for (int i = 0; i < sh.rounds; ++i) {
            const int r = row0 + i * step;
            const bool live = r < rows;
            Cols<V> p[NC][2], g[BWD ? NC : 1][2];
            auto sq = Cols<V>::all(0.0f), hx = sq;
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    p[n][k].from(nx[n][k]);
                    if constexpr (BWD) g[n][k].from(ng[n][k]);
#pragma unroll
                    for (int e = 0; e < N; ++e) sq = fma2(p[n][k].v[e], p[n][k].v[e], sq);
                }
            if (i + 1 < sh.rounds)
                fetch(t, r + step);
            else
                fetch(after, row0);
            if (i == 0 && at == 0) angles(then, angle + 2 * (buffer ^ 1) * sh.batch * pairs);
            if constexpr (BWD) {
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    const Chunks c(a, lane + n * sh.lanes);
                    if (c.turned) rotate<V, PAIRS, true>(g[n][0], g[n][1], cs_at + c.pair, cs_at + pairs + c.pair);
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < N; ++e) hx = fma2(mul2(g[n][k].v[e], wt[n][k].v[e]), p[n][k].v[e], hx);
                }
            }
            float square = sum2(sq), dot = sum2(hx);
            for (int m = sh.lanes >> 1; m >= 1; m >>= 1) {
                square += __shfl_xor_sync(0xffffffffu, square, m);
                if (BWD) dot += __shfl_xor_sync(0xffffffffu, dot, m);
            }
            if (!live) continue;
            // the reciprocal root by one step of Newton's from the approximate one
            const float var = fmaf(square, inv_d, a.eps), y0 = rsqrtf(var);
            const float step1 = y0 * fmaf(-0.5f * (var * y0), y0, 1.5f);
            const float rstd = !normed ? 1.0f : step1 == step1 ? step1 : y0;  // y0 is 0 or infinite
            const float along = normed ? -dot * rstd * rstd * inv_d : 0.0f;  // -mean(h xh) rstd, that x takes
            const auto r2 = Cols<V>::all(rstd), along2 = Cols<V>::all(along);
            T* out = wanted ? bo.at(a.out[which], tk, r - row0) : nullptr;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                if (lane + n * sh.lanes >= chunks) continue;
                const Chunks c(a, lane + n * sh.lanes);
                if (normed) {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < N; ++e) {
                            auto& x = p[n][k].v[e];
                            const auto w = wt[n][k].v[e];
                            if constexpr (BWD) {
                                auto& y = g[n][k].v[e];
                                dw[n][k].v[e] = fma2(y, mul2(x, r2), dw[n][k].v[e]);
                                y = mul2(r2, fma2(x, along2, mul2(y, w)));
                            } else {
                                x = mul2(mul2(x, r2), w);
                            }
                        }
                }
                if constexpr (BWD) {
                    if (out) {
                        g[n][0].store(out + c.c0);
                        g[n][1].store(out + c.c1);
                    }
                } else {
                    if (c.turned) rotate<V, PAIRS, false>(p[n][0], p[n][1], cs_at + c.pair, cs_at + pairs + c.pair);
                    p[n][0].store(out + c.c0);
                    p[n][1].store(out + c.c1);
                }
            }
        }
        at = more ? at + 1 : 0;
        buffer ^= !more;
        t = after;
    }
    if constexpr (BWD) {
        // the CTA's rows joined in the order of their groups
        float* part = angle + 4 * sh.batch * pairs;
        const int all = sh.slots[0] + sh.slots[1];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            if (lane + n * sh.lanes >= chunks || slot >= all) continue;
            const Chunks c(a, lane + n * sh.lanes);
            dw[n][0].store(part + slot * a.D + c.c0);
            dw[n][1].store(part + slot * a.D + c.c1);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * a.D; i += blockDim.x) {
            const int k = i / a.D, c = i % a.D;
            if (!a.sums[k]) continue;
            float v = 0.0f;
            for (int r = k ? sh.slots[0] : 0; r < (k ? all : sh.slots[0]); ++r) v += part[r * a.D + c];
            a.sums[k][static_cast<int64_t>(blockIdx.x) * a.D + c] = v;
        }
    }
}

template <typename T, bool BWD> qsml_status_t launch(Context* ctx, const RotaryArgs& a, const Shape& h, unsigned grid) {
    cudaError_t e = cudaSuccess;
    const bool one = a.D / (2 * h.vec) <= 32, two = a.D / (2 * h.vec) <= 64;
    auto go = [&](auto kernel) {
        e = launch_pdl(kernel, dim3(grid), dim3(h.threads), h.smem, ctx->stream, a, h);
    };
    auto pairing = [&](auto pairs) {
        constexpr bool P = decltype(pairs)::value;
        constexpr int FULL = 16 / sizeof(T);
        if (h.vec == FULL) {
            if constexpr (sizeof(T) == 2)
                go(k_norm_rotary<T, FULL, 1, P, BWD>);
            else
                one ? go(k_norm_rotary<T, FULL, 1, P, BWD>) : go(k_norm_rotary<T, FULL, 2, P, BWD>);
        } else if (h.vec == 2) {
            one ? go(k_norm_rotary<T, 2, 1, P, BWD>) : two ? go(k_norm_rotary<T, 2, 2, P, BWD>) : go(k_norm_rotary<T, 2, 4, P, BWD>);
        } else {
            one ? go(k_norm_rotary<T, 1, 1, P, BWD>) : two ? go(k_norm_rotary<T, 1, 2, P, BWD>) : go(k_norm_rotary<T, 1, 8, P, BWD>);
        }
    };
    a.pairs ? pairing(std::true_type()) : pairing(std::false_type());
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
    if (dq->B && dq->S > INT32_MAX / dq->B) return fail(ctx, QSML_E_UNSUPPORTED, op, "too many tokens");
    a->S = static_cast<int>(dq->S);
    a->T = static_cast<int>(dq->B * dq->S);
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

int64_t most_ctas(Context* ctx, const Shape& h) { return static_cast<int64_t>(ctx->num_sms) * (h.threads <= 256 ? 8 : 4); }

// All of a token's rows at once, or even shares of them.
Shape shape_of(Context* ctx, const RotaryArgs& a, int es, bool backward) {
    Shape h;
    h.vec = chunk_of(a, es, backward);
    const int chunks = a.D / (2 * h.vec);
    h.lanes = 1;
    while (h.lanes < chunks && h.lanes < 32) h.lanes *= 2;
    h.rounds = 1;
    for (;; ++h.rounds) {
        for (int k = 0; k < 2; ++k) h.slots[k] = (a.H[k] + h.rounds - 1) / h.rounds;
        if (static_cast<int64_t>(h.slots[0] + h.slots[1]) * h.lanes <= most_threads(backward)) break;
    }
    const int all = h.slots[0] + h.slots[1];
    h.threads = (all * h.lanes + 31) / 32 * 32;
    // a batch has an angle for every lane, where there are that many tokens for every CTA: the angles
    // of a token at a time, by two of ten warps, keep the others waiting
    const int64_t tokens = a.T / std::max<int64_t>(1, most_ctas(ctx, h));
    h.batch = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(std::min(8, h.threads / (a.rot / 2)), tokens)));
    h.smem = 2 * sizeof(float) * a.rot * h.batch + (backward ? sizeof(float) * all * a.D : 0);
    return h;
}

// A batch a CTA, or as many CTAs as fill the device.
unsigned grid_of(Context* ctx, const RotaryArgs& a, const Shape& h) {
    return static_cast<unsigned>(std::min<int64_t>((static_cast<int64_t>(a.T) + h.batch - 1) / h.batch, most_ctas(ctx, h)));
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
    const Shape h = shape_of(C_, a, dtype_size(q->dtype), false);
    const unsigned grid = grid_of(C_, a, h);
    return q->dtype == QSML_F16 ? launch<__half, false>(C_, a, h, grid) : launch<float, false>(C_, a, h, grid);
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
    const Shape h = shape_of(C_, a, dtype_size(q->dtype), true);
    const unsigned grid = grid_of(C_, a, h);
    Workspace ws(C_);
    ColumnSum sums[2];
    for (int i = 0; i < 2; ++i) {
        if (!dw[i] || !a.H[i]) continue;
        void* p = nullptr;
        QSML_TRY_STATUS(ws.get(sizeof(float) * a.D * grid, &p));
        a.sums[i] = static_cast<float*>(p);
        sums[i] = ColumnSum{a.sums[i], dw[i]->data, dw[i]->dtype};
    }
    QSML_TRY_STATUS((q->dtype == QSML_F16 ? launch<__half, true>(C_, a, h, grid) : launch<float, true>(C_, a, h, grid)));
    return finish_column_sums(C_, sums[0], sums[1], grid, a.D);
} QSML_NO_THROW
