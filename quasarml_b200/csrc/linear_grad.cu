// Gradients of the linear layers with respect to their products, and the
// biases' gradients: one pass over dy and what the forward pass kept.
//   LINEAR: dz = dy act'(pre)            db = column sums of dz
//   DUAL:   dg = dy u act'(g), du = dy act(g), and the column sums of both
// dz goes to a workspace that the two products of the backward pass read (in the parts
// that the tensor cores take, see GradArgs); the sums are taken before it is rounded.
// Bound by HBM: LINEAR reads 2 and writes 1 element, DUAL reads 3 and writes 2 (binary16:
// 16384 x 2048 with gelu 38 us, 5.3 TB/s; DUAL 8192 x 5632 76 us, 6.1 TB/s).
#include "linear_grad.cuh"

namespace qsml {
namespace linear {
namespace {

// Eight consecutive elements as they were loaded, by the read-only path (no output
// of the call overlaps an input).
template <typename T> struct alignas(16) Raw8 {
    T v[8];
    __device__ void load(const T* p, int n, bool vec) {
        if (vec) {
            constexpr int Q = sizeof(T) * 8 / 16;
            uint4* d = reinterpret_cast<uint4*>(v);
#pragma unroll
            for (int q = 0; q < Q; ++q) d[q] = __ldg(reinterpret_cast<const uint4*>(p) + q);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : T(0.0f);
        }
    }
    __device__ P2 pair(int j) const {  // elements 2 j and 2 j + 1
        const float2 f = ld2(v + 2 * j);
        return pack(f.x, f.y);
    }
};

// A warp takes 256 columns (8 a lane), a CTA's 8 warps every 8th row of
// [blockIdx.y * chunk, + chunk).  A thread keeps its columns and sums them in
// registers; the warps' sums are added in warp order in shared memory.
template <typename T, bool DUAL, int ACT>
__global__ void __launch_bounds__(256) k_linear_dz(const __grid_constant__ GradArgs a, int64_t chunk, bool vec) {
    pdl_begin();
    constexpr int NO = DUAL ? 2 : 1;
    __shared__ float fold[NO][8][256 + 8];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 256 + lane * 8;
    const int n = a.N - col < 8 ? static_cast<int>(a.N - col) : 8;  // may be <= 0
    const int64_t r0 = blockIdx.y * chunk, r1 = r0 + chunk < a.M ? r0 + chunk : a.M;
    P2 sum[NO][4];
#pragma unroll
    for (int o = 0; o < NO; ++o)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[o][j].v = 0;
    if (n > 0) {
        // AHEAD rows in flight under the one at hand: as many as leave two CTAs a SM, three
        // LINEAR ones of binary16 (DUAL binary16 8192 x 5632: 88, 79, 76 us with 1, 2, 3;
        // binary32 8192 x 4096: 128 us with 1, 171 with 2)
        constexpr int AHEAD = sizeof(T) == 4 ? 1 : DUAL ? 3 : 2;
        constexpr bool PRE = DUAL || ACT != QSML_ACT_NONE;
        Raw8<T> ry[AHEAD + 1], rz[AHEAD + 1], ru[AHEAD + 1];
        auto load = [&](int64_t r, Raw8<T>& y, Raw8<T>& z, Raw8<T>& u) {
            if (r >= r1) return;
            y.load(static_cast<const T*>(a.dy) + r * a.dy_ld + col, n, vec);
            if constexpr (PRE) z.load(static_cast<const T*>(a.pre[0]) + r * a.N + col, n, vec);
            if constexpr (DUAL) u.load(static_cast<const T*>(a.pre[1]) + r * a.N + col, n, vec);
        };
        auto work = [&](int64_t r, const Raw8<T>& y, const Raw8<T>& z, const Raw8<T>& u) {
            // elements past the row's end were loaded as 0 and so end as 0
            P2 d[NO][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (!PRE) {
                    d[0][j] = y.pair(j);
                } else {
                    P2 value;
                    const P2 g = act_grad2<T>(ACT, z.pair(j), value);
                    if constexpr (DUAL) {
                        d[0][j] = mul2(mul2(y.pair(j), u.pair(j)), g);
                        d[1][j] = mul2(y.pair(j), value);
                    } else {
                        d[0][j] = mul2(y.pair(j), g);
                    }
                }
            }
#pragma unroll
            for (int o = 0; o < NO; ++o) {
                if (a.dz[o]) {
                    float f[8];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 e = unpack(d[o][j]);
                        f[2 * j] = e.x;
                        f[2 * j + 1] = e.y;
                    }
                    if (a.plane) {
                        uint16_t* to = static_cast<uint16_t*>(a.dz[o]) + r * a.pitch + col;
                        if constexpr (sizeof(T) == 4) split8(f, to, a.plane);
                        else halve8(f, reinterpret_cast<__half*>(to), a.plane);
                    } else {
                        store8(static_cast<T*>(a.dz[o]) + r * a.pitch + col, n, n == 8, f);
                    }
                }
                if (a.partial) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum[o][j] = add2(sum[o][j], d[o][j]);
                }
            }
        };
        int64_t r = r0 + w;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) load(r + 8 * i, ry[i], rz[i], ru[i]);
        while (r < r1) {
#pragma unroll
            for (int i = 0; i <= AHEAD; ++i) {
                if (r >= r1) break;
                const int to = (i + AHEAD) % (AHEAD + 1);
                load(r + 8 * AHEAD, ry[to], rz[to], ru[to]);
                work(r, ry[i], rz[i], ru[i]);
                r += 8;
            }
        }
    }
    if (!a.partial) return;
#pragma unroll
    for (int o = 0; o < NO; ++o)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 e = unpack(sum[o][j]);
            fold[o][w][lane * 8 + 2 * j] = e.x;
            fold[o][w][lane * 8 + 2 * j + 1] = e.y;
        }
    __syncthreads();
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (c >= a.N) return;
#pragma unroll
    for (int o = 0; o < NO; ++o) {
        float s = fold[o][0][threadIdx.x];
        for (int k = 1; k < 8; ++k) s = __fadd_rn(s, fold[o][k][threadIdx.x]);
        a.partial[(static_cast<int64_t>(o) * gridDim.y + blockIdx.y) * a.N + c] = s;
    }
}

template <typename T, bool DUAL> qsml_status_t launch(Context* ctx, const GradArgs& given) {
    GradArgs a = given;
    const int64_t tiles = (a.N + 255) / 256;
    // about eight CTAs an SM, at least 2 rows a warp (8 left most SMs without a CTA at
    // 515 x 1366: 23 us)
    int64_t parts = (8 * ctx->num_sms + tiles - 1) / tiles;
    const int64_t most = (a.M + 15) / 16;
    if (parts > most) parts = most;
    const int64_t chunk = (a.M + parts - 1) / parts;
    parts = (a.M + chunk - 1) / chunk;
    Workspace ws(ctx);
    const bool sums = a.db[0].out || a.db[1].out;
    void* partial = nullptr;
    if (sums) QSML_TRY_STATUS(ws.get(static_cast<size_t>(DUAL ? 2 : 1) * parts * a.N * sizeof(float), &partial));
    a.partial = static_cast<float*>(partial);
    bool vec = a.N % 8 == 0 && a.dy_ld % 8 == 0 && aligned16(a.dy);
    for (int i = 0; i < 2; ++i) vec = vec && (!a.pre[i] || aligned16(a.pre[i]));
    auto kernel = k_linear_dz<T, DUAL, QSML_ACT_NONE>;
    switch (a.act) {
        case QSML_ACT_RELU: kernel = k_linear_dz<T, DUAL, QSML_ACT_RELU>; break;
        case QSML_ACT_GELU: kernel = k_linear_dz<T, DUAL, QSML_ACT_GELU>; break;
        case QSML_ACT_SILU: kernel = k_linear_dz<T, DUAL, QSML_ACT_SILU>; break;
        case QSML_ACT_SIGMOID: kernel = k_linear_dz<T, DUAL, QSML_ACT_SIGMOID>; break;
    }
    const cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(parts)),
                                     dim3(256), 0, ctx->stream, a, chunk, vec);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_linear_dz");
    QSML_TRY_STATUS(after_launch(ctx, "k_linear_dz"));
    if (!sums) return QSML_OK;
    ColumnSum s0 = a.db[0], s1 = a.db[1];
    s0.partial = a.partial;
    s1.partial = a.partial + parts * a.N;
    return finish_column_sums(ctx, s0, s1, parts, a.N);
}

}  // namespace

template <typename T> qsml_status_t run_grad(Context* ctx, const GradArgs& a, bool dual) {
    return dual ? launch<T, true>(ctx, a) : launch<T, false>(ctx, a);
}
template qsml_status_t run_grad<float>(Context*, const GradArgs&, bool);
template qsml_status_t run_grad<__half>(Context*, const GradArgs&, bool);

}  // namespace linear
}  // namespace qsml
