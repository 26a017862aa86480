// What the kernels of the linear layers share: the problem they are given and
// the arithmetic behind the products (bias, activation, residual).
//
//   out = sum over segments s of A_s B_s          (LINEAR)
//   (g, u) = (A B_0, A B_1)                        (DUAL: two products of one A)
// LINEAR:  z = out + bias;  pre = z;  y = act(z) + residual
// DUAL:    g += bias_0, u += bias_1;  pre_0 = g, pre_1 = u;  y = act(g) u
// where every output that is null is left out.  All of it is binary32, each
// output rounded once.
#pragma once

#include "packed.cuh"
#include "workspace.cuh"

namespace qsml {
namespace linear {

// A matrix as given: element (r, c) at p + r * rs + c * cs (elements).  plane > 0:
// values in parts for the tensor cores, `plane` elements apart, one of the strides
// being 1 and the other a multiple of 8: binary32 as three bf16 (split8), or binary32
// values of a binary16 problem as two binary16 (halve8).
struct Mat {
    const void* p = nullptr;
    int64_t rows = 0, cols = 0, rs = 0, cs = 0, plane = 0;
    Mat t() const { return Mat{p, cols, rows, cs, rs, plane}; }
};

// Elements between the rows of a 16-bit workspace matrix: whole 128-byte lines, so
// that a 128-byte box row is one (a pitch of 1032 doubled the L2 traffic).
inline int64_t line_pitch(int64_t cols) { return (cols + 63) / 64 * 64; }

struct Epilogue {
    const float* scale = nullptr;  // binary16: the products are multiplied by it, a power of two; null: by 1
    const void* bias[2] = {nullptr, nullptr};
    int bias_f32 = 1;              // else the dtype of the outputs
    int act = QSML_ACT_NONE;
    const void* residual = nullptr;
    int64_t res_ld = 0;            // elements between residual rows
    void* pre[2] = {nullptr, nullptr};
    void* y = nullptr;             // y and pre: rows of N elements
    int64_t N = 0;
    int vec = 0;                   // 1: groups of 8 columns are whole and 16-byte aligned everywhere; 2: pairs are
                                   // whole and aligned; 0: neither
};

struct Problem {
    int64_t M = 0, N = 0, K = 0;
    int segments = 1;              // 2: a[0] b[0] + a[1] b[1]
    bool dual = false;             // a[0] b[0] and a[0] b[1]
    Mat a[2], b[2];
    Epilogue e;
};

// CUDA-core products, binary32 fma with k ascending: any strides, any size.
template <typename T> qsml_status_t run_simt(Context* ctx, const Problem& p);

// Binary32 products of at most 16 rows (8 for a dual product) with weights that are
// contiguous along one dim: whether p is one, and its kernel (linear_few.cu).
bool few_rows(const Problem& p);
qsml_status_t run_few(Context* ctx, const Problem& p);

// Tensor-core products (linear_tc.cu), any strides, alignment and size with
// K > 0: binary16, or binary32 as three bf16 parts.  The operands of all n (at
// most 2) problems that have to be copied are copied in one launch.
qsml_status_t run_tc(Context* ctx, const Problem* const* p, int n, bool f32);

// ---- arithmetic shared by the kernels --------------------------------------------
__device__ __forceinline__ float ld1(const float* p) { return *p; }
__device__ __forceinline__ float ld1(const __half* p) { return __half2float(*p); }

constexpr float kGeluS = 0.7978845608f, kGeluC = 0.044715f;  // the constants of QSML_UN_GELU
constexpr float kLog2e = 1.4426950408889634f;

// Activations are computed two values at a time (packed.cuh): one by one they took 29
// instructions an element in the gradient's pass, which bound it.

// 1 / (1 + exp(-z)); 0 where exp(-z) overflows.  Binary32 results take expf and a
// correctly rounded reciprocal.  Binary16 ones take 2^t and 1/d of the hardware
// (2 ulp and 1 ulp; t = -z log2(e) is off by 2^-24 |t|): far below half a step of
// binary16, and a third of the instructions, which bounded the epilogue and the
// gradient's pass.
template <typename T> __device__ __forceinline__ P2 act_sigmoid2(P2 z) {
    if constexpr (sizeof(T) == 2) {
        const float2 t = unpack(mul2(both(-kLog2e), z));
        float2 e, p;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
        const float2 d = unpack(add2(both(1.0f), pack(e.x, e.y)));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(p.x) : "f"(d.x));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(p.y) : "f"(d.y));
        return pack(p.x, p.y);
    } else {
        const float2 f = unpack(z);
        return pack(__frcp_rn(__fadd_rn(1.0f, expf(-f.x))), __frcp_rn(__fadd_rn(1.0f, expf(-f.y))));
    }
}
// act of two values.  gelu: 0.5 z (1 + tanh v) = z sigmoid(2 v), v = s (z + c z^3).
template <typename T> __device__ __forceinline__ P2 act_value2(int act, P2 z) {
    switch (act) {
        case QSML_ACT_RELU: {
            const float2 f = unpack(z);
            return pack(f.x != f.x ? f.x : (f.x > 0.0f ? f.x : 0.0f), f.y != f.y ? f.y : (f.y > 0.0f ? f.y : 0.0f));
        }
        case QSML_ACT_GELU: {
            const P2 q = mul2(z, z), s2 = both(2.0f * kGeluS);
            return mul2(z, act_sigmoid2<T>(mul2(mul2(s2, z), fma2(both(kGeluC), q, both(1.0f)))));
        }
        case QSML_ACT_SILU: return mul2(z, act_sigmoid2<T>(z));
        case QSML_ACT_SIGMOID: return act_sigmoid2<T>(z);
    }
    return z;
}

// act of N values, one branch for all of them
template <typename T, int N> __device__ __forceinline__ void act_all(int act, float (&z)[N]) {
    static_assert(N % 2 == 0, "pairs");
    auto all = [&](auto kind) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 f = unpack(act_value2<T>(kind.value, pack(z[i], z[i + 1])));
            z[i] = f.x;
            z[i + 1] = f.y;
        }
    };
    switch (act) {
        case QSML_ACT_RELU: all(std::integral_constant<int, QSML_ACT_RELU>{}); break;
        case QSML_ACT_GELU: all(std::integral_constant<int, QSML_ACT_GELU>{}); break;
        case QSML_ACT_SILU: all(std::integral_constant<int, QSML_ACT_SILU>{}); break;
        case QSML_ACT_SIGMOID: all(std::integral_constant<int, QSML_ACT_SIGMOID>{}); break;
    }
}

// act(z) and its derivative.  With p the sigmoid:
//   silu' = p + z p (1 - p);  sigmoid' = p (1 - p);
//   gelu' = p + z p (1 - p) 2 v',  2 v' = 2 s (1 + 3 c z^2).
// sigmoid' is even: taken at -|z|, where p is the small factor and 1 - p loses nothing (at
// z = 12 1 - p has 7 bits left).  In the others p itself is beside the product there.
template <typename T> __device__ __forceinline__ P2 act_grad2(int act, P2 z, P2& value) {
    const P2 one = both(1.0f);
    switch (act) {
        case QSML_ACT_RELU: {
            const float2 f = unpack(z);
            value = act_value2<T>(QSML_ACT_RELU, z);
            return pack(f.x != f.x ? f.x : (f.x > 0.0f ? 1.0f : 0.0f), f.y != f.y ? f.y : (f.y > 0.0f ? 1.0f : 0.0f));
        }
        case QSML_ACT_GELU: {
            P2 q = mul2(z, z);
            const P2 s2 = both(2.0f * kGeluS);
            if constexpr (sizeof(T) == 4) {  // from 1e19 on z z is infinite, and 0 times that no number
                const float2 f = unpack(q);
                q = pack(fminf(f.x, 0x1p96f), fminf(f.y, 0x1p96f));
            }
            const P2 p = act_sigmoid2<T>(mul2(mul2(s2, z), fma2(both(kGeluC), q, one)));
            value = mul2(z, p);
            const P2 dv = mul2(s2, fma2(both(3.0f * kGeluC), q, one));
            return fma2(mul2(value, fma2(p, both(-1.0f), one)), dv, p);
        }
        case QSML_ACT_SILU: {
            const P2 p = act_sigmoid2<T>(z);
            value = mul2(z, p);
            return fma2(value, fma2(p, both(-1.0f), one), p);
        }
        case QSML_ACT_SIGMOID: {
            const float2 f = unpack(z);
            const P2 p = act_sigmoid2<T>(pack(-fabsf(f.x), -fabsf(f.y))), q = fma2(p, both(-1.0f), one);
            const float2 pf = unpack(p), qf = unpack(q);
            value = pack(f.x > 0.0f ? qf.x : pf.x, f.y > 0.0f ? qf.y : pf.y);
            return mul2(p, q);
        }
    }
    value = z;
    return one;
}

// Two neighbours, aligned together.
__device__ __forceinline__ float2 ld2(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 ld2(const __half* p) { return __half22float2(*reinterpret_cast<const __half2*>(p)); }
__device__ __forceinline__ void st2(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void st2(__half* p, float a, float b) {
    *reinterpret_cast<__half2*>(p) = __floats2half2_rn(a, b);
}

// 8 consecutive elements of a row to binary32 and back; n of them are inside
// (vec as in Epilogue).
template <typename T> __device__ __forceinline__ void load8(const T* p, int n, int vec, float (&v)[8]) {
    if (vec == 1) {
        if constexpr (sizeof(T) == 2) {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(h[i]);
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        } else {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        }
    } else if (vec == 2) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float2 f = i < n ? ld2(p + i) : make_float2(0.0f, 0.0f);
            v[i] = f.x;
            v[i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? ld1(p + i) : 0.0f;
    }
}
// The same through the read-only path, for inputs that nothing writes meanwhile.
template <typename T> __device__ __forceinline__ void ldg8(const T* p, int n, bool vec, float (&v)[8]) {
    if (vec) {
        if constexpr (sizeof(T) == 2) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
            const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(h[i]);
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        } else {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        }
    } else {
        load8(p, n, false, v);
    }
}
template <typename T> __device__ __forceinline__ void store8(T* p, int n, int vec, const float (&v)[8]) {
    if (vec == 2) {
#pragma unroll
        for (int i = 0; i < 8; i += 2)
            if (i < n) st2(p + i, v[i], v[i + 1]);
        return;
    }
    if constexpr (sizeof(T) == 2) {
        if (vec) {
            uint4 u;
            __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            *reinterpret_cast<uint4*>(p) = u;
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = __float2half_rn(v[i]);
    } else {
        if (vec) {
            reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = v[i];
    }
}

// x = x0 + x1 + x2 in bf16, exactly: each part the upper 8 bits of what is left,
// truncated (a bf16 is the upper half of a binary32).  Below 2^-110 the last part
// may fall under the smallest number and is cut.  Infinities and NaN are all x0.
__device__ __forceinline__ void split3(float x, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
    const uint32_t b = __float_as_uint(x), top = b & 0xffff0000u;
    if ((b & 0x7f800000u) == 0x7f800000u) {
        p0 = (b >> 16) | ((b & 0xffffu) ? 0x40u : 0u);  // a NaN stays one
        p1 = p2 = 0;
        return;
    }
    const float r1 = __fsub_rn(x, __uint_as_float(top));
    const uint32_t t1 = __float_as_uint(r1) & 0xffff0000u;
    const float r2 = __fsub_rn(r1, __uint_as_float(t1));
    p0 = top >> 16;
    p1 = t1 >> 16;
    p2 = __float_as_uint(r2) >> 16;
}
// Eight of them to three rows of bf16, `plane` elements apart (16-byte aligned).
__device__ __forceinline__ void split8(const float (&v)[8], uint16_t* dst, int64_t plane) {
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t a[3], b[3];
        split3(v[2 * i], a[0], a[1], a[2]);
        split3(v[2 * i + 1], b[0], b[1], b[2]);
#pragma unroll
        for (int p = 0; p < 3; ++p) w[p][i] = a[p] | (b[p] << 16);
    }
#pragma unroll
    for (int p = 0; p < 3; ++p)
        *reinterpret_cast<uint4*>(dst + p * plane) = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
}

// x = h0 + h1 + (below 2^-22 |x|, or 2^-25), h0 and h1 binary16; an x beyond their
// range is h0 = infinity and h1 = 0.  Eight of them to two rows, `plane` elements apart.
__device__ __forceinline__ void halve8(const float (&v)[8], __half* dst, int64_t plane) {
    float hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        hi[i] = __half2float(__float2half_rn(v[i]));
        lo[i] = fabsf(hi[i]) < 65536.0f ? __fsub_rn(v[i], hi[i]) : 0.0f;
    }
    store8(dst, 8, true, hi);
    store8(dst + plane, 8, true, lo);
}

// The biases of columns col .. col + 7 (0 where there is none), for finish8.
template <typename T, bool DUAL>
__device__ __forceinline__ void bias8(const Epilogue& e, int64_t col, float (&b)[DUAL ? 2 : 1][8]) {
    const int n = e.N - col < 8 ? static_cast<int>(e.N - col) : 8;
#pragma unroll
    for (int w = 0; w < (DUAL ? 2 : 1); ++w) {
        if (!e.bias[w]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) b[w][i] = 0.0f;
        } else if (e.bias_f32) {
            load8(static_cast<const float*>(e.bias[w]) + col, n, e.vec == 1, b[w]);
        } else {
            load8(static_cast<const T*>(e.bias[w]) + col, n, e.vec == 1, b[w]);
        }
    }
}

// What Epilogue::scale points to.
template <typename T> __device__ __forceinline__ float scale_of(const Epilogue& e) {
    if constexpr (sizeof(T) == 4) return 1.0f;
    return e.scale ? *e.scale : 1.0f;
}

// Columns col .. col + 7 of `row` from their products (u: DUAL only), which are
// multiplied by `scale`, to the outputs.  col is a multiple of 8; columns from N on are
// not written.
template <typename T, bool DUAL>
__device__ __forceinline__ void finish8(const Epilogue& e, int64_t row, int64_t col, const float (&b)[DUAL ? 2 : 1][8],
                                        float (&z)[8], float (&u)[8], float scale = 1.0f) {
    const int n = e.N - col < 8 ? static_cast<int>(e.N - col) : 8;
    const int64_t at = row * e.N + col;
    float r[8];
    if constexpr (!DUAL) {  // first, so that it is in flight under the rest
        if (e.residual) load8(static_cast<const T*>(e.residual) + row * e.res_ld + col, n, e.vec, r);
    }
    if (scale != 1.0f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            z[i] = __fmul_rn(z[i], scale);
            if constexpr (DUAL) u[i] = __fmul_rn(u[i], scale);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        z[i] = __fadd_rn(z[i], b[0][i]);
        if constexpr (DUAL) u[i] = __fadd_rn(u[i], b[DUAL ? 1 : 0][i]);
    }
    if (e.pre[0]) store8(static_cast<T*>(e.pre[0]) + at, n, e.vec, z);
    if constexpr (DUAL) {
        if (e.pre[1]) store8(static_cast<T*>(e.pre[1]) + at, n, e.vec, u);
    }
    if (!e.y) return;
    act_all<T>(e.act, z);
    if constexpr (DUAL) {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = __fmul_rn(z[i], u[i]);
    } else if (e.residual) {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = __fadd_rn(z[i], r[i]);
    }
    store8(static_cast<T*>(e.y) + at, n, e.vec, z);
}

template <typename T> __device__ __forceinline__ float bias1(const Epilogue& e, int which, int64_t col) {
    if (!e.bias[which]) return 0.0f;
    return e.bias_f32 ? static_cast<const float*>(e.bias[which])[col] : ld1(static_cast<const T*>(e.bias[which]) + col);
}
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(__half* p, float v) { *p = __float2half_rn(v); }

}  // namespace linear
}  // namespace qsml
