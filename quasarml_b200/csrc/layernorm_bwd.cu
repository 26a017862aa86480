// Backward pass of the layer norm over the last dim.  With
//   xh = (x - mean) rstd,  h = dy gamma,
//   c1 = mean_c(h),        c2 = mean_c(h xh)          (means along the row)
// the gradients are
//   dx = rstd (h - c1 - xh c2),   dgamma_c = sum_r dy xh,   dbeta_c = sum_r dy.
// The forward pass keeps nothing for it: mean and rstd are computed again from
// the row, which has to be read for xh anyway.  The reference has no layer
// norm and no gradients.
//
// k_layer_norm_bwd: a CTA (or, for narrow rows, a warp) holds a row of x and dy
// in registers, so both are read once and dx is written once (3 elements of
// traffic, the floor).  Row sums take two steps: the row sum, then together
// the squared deviations, sum(h) and sum(h (x - mean)), all about the mean, so
// nothing is lost by cancellation.  A thread keeps its columns for every row
// it meets and so sums dgamma and dbeta in registers (binary32); the CTAs'
// sums are joined by k_column_finish in a fixed order.
// k_layer_norm_bwd_rows + k_layer_norm_bwd_cols: rows wider than the registers
// hold, in two kernels (5 elements of traffic and the row statistics).
#include "workspace.cuh"

namespace qsml {
namespace {

template <typename T, int N> struct alignas(N * sizeof(T)) Vec {
    T v[N];
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f(float v, __half& o) { o = __float2half_rn(v); }

__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}

// Sums of `n` values over the threads that share a row: a warp (WARP) or the
// CTA, every thread ending with the same bits.  `slot` (n x 32 floats) is not
// written again before every thread has read it: callers alternate two.
template <bool WARP, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* slot) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_add(v[i]);
    if constexpr (!WARP) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) slot[i * 32 + w] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = warp_add(lane < nw ? slot[i * 32 + lane] : 0.0f);
    }
}

// PV elements a load, NV loads a thread.  partial: [gridDim.x][cols] of dgamma
// followed by the same of dbeta (null: not wanted).  dx may be null.
template <typename T, typename GT, int PV, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 512)
    k_layer_norm_bwd(const T* __restrict__ x, const GT* __restrict__ gamma, const T* __restrict__ dy,
                     T* __restrict__ dx, float* __restrict__ partial, int64_t rows, int cols, float eps) {
    pdl_begin();
    constexpr int E = NV * PV;
    using V = Vec<T, PV>;
    __shared__ float slots[4 * 32];
    extern __shared__ float fold[];  // WARP: the warps' column sums, [2][cols]
    const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int th = WARP ? 32 : blockDim.x;
    const int per = WARP ? blockDim.x >> 5 : 1;  // rows a CTA has at a time
    const int packs = cols / PV;
    float g[E], sg[E], sb[E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int p = t + i * th;
#pragma unroll
        for (int e = 0; e < PV; ++e) {
            g[i * PV + e] = p < packs ? to_f(gamma[p * PV + e]) : 0.0f;
            sg[i * PV + e] = 0.0f;
            sb[i * PV + e] = 0.0f;
        }
    }
    const float inv_n = __frcp_rn(static_cast<float>(cols));
    const int64_t step = static_cast<int64_t>(gridDim.x) * per;
    int64_t row = static_cast<int64_t>(blockIdx.x) * per + (WARP ? threadIdx.x >> 5 : 0);
    V nx[NV], ny[NV];
    auto load = [&](int64_t r) {
        const V* xr = reinterpret_cast<const V*>(x + r * cols);
        const V* yr = reinterpret_cast<const V*>(dy + r * cols);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int p = t + i * th;
            if (p < packs) {
                nx[i] = xr[p];
                ny[i] = yr[p];
            }
        }
    };
    if (row < rows) load(row);
    for (; row < rows; row += step) {
        float d[E], y[E];
        float s1[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool in = t + i * th < packs;
#pragma unroll
            for (int e = 0; e < PV; ++e) {
                d[i * PV + e] = in ? to_f(nx[i].v[e]) : 0.0f;
                y[i * PV + e] = in ? to_f(ny[i].v[e]) : 0.0f;
                s1[0] = __fadd_rn(s1[0], d[i * PV + e]);
            }
        }
        if (row + step < rows) load(row + step);  // in flight while this row is reduced
        row_sums<WARP>(s1, slots);
        const float mean = __fmul_rn(s1[0], inv_n);
        float s3[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool in = t + i * th < packs;
#pragma unroll
            for (int e = 0; e < PV; ++e) {
                const int k = i * PV + e;
                d[k] = in ? __fsub_rn(d[k], mean) : 0.0f;
                const float h = __fmul_rn(y[k], g[k]);
                s3[0] = __fmaf_rn(d[k], d[k], s3[0]);
                s3[1] = __fadd_rn(s3[1], h);
                s3[2] = __fmaf_rn(h, d[k], s3[2]);
            }
        }
        row_sums<WARP>(s3, slots + 32);
        const float rstd = rsqrtf(__fmaf_rn(s3[0], inv_n, eps));
        // dx = rstd h - rstd c1 - d (rstd^2 c2),  c2 = mean(h d) rstd
        const float a = __fmul_rn(__fmul_rn(s3[1], inv_n), rstd);
        const float b = __fmul_rn(__fmul_rn(__fmul_rn(s3[2], inv_n), rstd), __fmul_rn(rstd, rstd));
        V out[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < PV; ++e) {
                const int k = i * PV + e;
                const float h = __fmul_rn(y[k], g[k]);
                from_f(__fmaf_rn(h, rstd, -__fmaf_rn(d[k], b, a)), out[i].v[e]);
                sg[k] = __fmaf_rn(y[k], __fmul_rn(d[k], rstd), sg[k]);
                sb[k] = __fadd_rn(sb[k], y[k]);
            }
        if (dx) {
            V* dr = reinterpret_cast<V*>(dx + row * cols);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (t + i * th < packs) dr[t + i * th] = out[i];
        }
    }
    if (!partial) return;
    float* pg = partial + static_cast<int64_t>(blockIdx.x) * cols;
    float* pb = pg + static_cast<int64_t>(gridDim.x) * cols;
    if constexpr (WARP) {
        // the warps' sums, one warp after another
        for (int w = 0; w < per; ++w) {
            if (static_cast<int>(threadIdx.x >> 5) == w) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (t + i * th < packs)
#pragma unroll
                        for (int e = 0; e < PV; ++e) {
                            const int c = (t + i * th) * PV + e, k = i * PV + e;
                            fold[c] = w ? __fadd_rn(fold[c], sg[k]) : sg[k];
                            fold[cols + c] = w ? __fadd_rn(fold[cols + c], sb[k]) : sb[k];
                        }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < cols; c += blockDim.x) {
            pg[c] = fold[c];
            pb[c] = fold[cols + c];
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (t + i * th < packs)
#pragma unroll
                for (int e = 0; e < PV; ++e) {
                    const int c = (t + i * th) * PV + e;
                    pg[c] = sg[i * PV + e];
                    pb[c] = sb[i * PV + e];
                }
    }
}

// Rows of any width, a CTA a row in three sweeps over global memory (L2 holds a
// row between them); leaves the row's mean and rstd for the column kernel.
template <typename T, typename GT>
__global__ void __launch_bounds__(512)
    k_layer_norm_bwd_rows(const T* __restrict__ x, const GT* __restrict__ gamma, const T* __restrict__ dy,
                          T* __restrict__ dx, float2* __restrict__ stats, int64_t rows, int64_t cols, float eps) {
    pdl_begin();
    __shared__ float slots[4 * 32];
    const float inv_n = __frcp_rn(static_cast<float>(cols));
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row * cols;
        const T* yr = dy + row * cols;
        float s1[1] = {0.0f};
        for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) s1[0] = __fadd_rn(s1[0], to_f(xr[c]));
        row_sums<false>(s1, slots);
        const float mean = __fmul_rn(s1[0], inv_n);
        float s3[3] = {0.0f, 0.0f, 0.0f};
        for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
            const float d = __fsub_rn(to_f(xr[c]), mean), h = __fmul_rn(to_f(yr[c]), to_f(gamma[c]));
            s3[0] = __fmaf_rn(d, d, s3[0]);
            s3[1] = __fadd_rn(s3[1], h);
            s3[2] = __fmaf_rn(h, d, s3[2]);
        }
        row_sums<false>(s3, slots + 32);
        const float rstd = rsqrtf(__fmaf_rn(s3[0], inv_n, eps));
        if (stats && threadIdx.x == 0) stats[row] = make_float2(mean, rstd);
        if (!dx) continue;
        const float a = __fmul_rn(__fmul_rn(s3[1], inv_n), rstd);
        const float b = __fmul_rn(__fmul_rn(__fmul_rn(s3[2], inv_n), rstd), __fmul_rn(rstd, rstd));
        for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
            const float d = __fsub_rn(to_f(xr[c]), mean), h = __fmul_rn(to_f(yr[c]), to_f(gamma[c]));
            from_f(__fmaf_rn(h, rstd, -__fmaf_rn(d, b, a)), dx[row * cols + c]);
        }
    }
}

// Column sums of dy xh and dy over the rows [blockIdx.y * chunk, + chunk): a
// thread a column.
template <typename T>
__global__ void __launch_bounds__(256)
    k_layer_norm_bwd_cols(const T* __restrict__ x, const T* __restrict__ dy, const float2* __restrict__ stats,
                          float* __restrict__ partial, int64_t rows, int64_t cols, int64_t chunk) {
    pdl_begin();
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (c >= cols) return;
    const int64_t r0 = blockIdx.y * chunk, r1 = r0 + chunk < rows ? r0 + chunk : rows;
    float sg = 0.0f, sb = 0.0f;
#pragma unroll 4
    for (int64_t r = r0; r < r1; ++r) {
        const float2 st = stats[r];
        const float y = to_f(dy[r * cols + c]);
        sg = __fmaf_rn(y, __fmul_rn(__fsub_rn(to_f(x[r * cols + c]), st.x), st.y), sg);
        sb = __fadd_rn(sb, y);
    }
    partial[blockIdx.y * cols + c] = sg;
    partial[(gridDim.y + static_cast<int64_t>(blockIdx.y)) * cols + c] = sb;
}

struct Args {
    const void *x, *gamma, *dy;
    void* dx;
    ColumnSum sg, sb;  // out pointers and dtypes
    int64_t rows, cols;
    float eps;
    bool sums() const { return sg.out || sb.out; }
};

qsml_status_t finish(Context* ctx, const Args& a, float* partial, int64_t parts) {
    ColumnSum g = a.sg, b = a.sb;
    g.partial = partial;
    b.partial = partial + parts * a.cols;
    return finish_column_sums(ctx, g, b, parts, a.cols);
}

template <typename T, typename GT, int PV, int NV, bool WARP>
qsml_status_t launch_bwd(Context* ctx, const Args& a, int th) {
    auto kernel = k_layer_norm_bwd<T, GT, PV, NV, WARP>;
    const int per = WARP ? 8 : 1;
    const int block = WARP ? 256 : th;
    const size_t smem = WARP && a.sums() ? static_cast<size_t>(a.cols) * 2 * sizeof(float) : 0;
    int per_sm = 0;
    QSML_TRY_STATUS(check_cuda(ctx, cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, block, smem),
                               "layer norm backward: occupancy"));
    int64_t grid = static_cast<int64_t>(ctx->num_sms) * (per_sm < 1 ? 1 : per_sm);
    const int64_t most = (a.rows + per - 1) / per;
    if (grid > most) grid = most;
    Workspace ws(ctx);
    void* partial = nullptr;
    if (a.sums()) QSML_TRY_STATUS(ws.get(static_cast<size_t>(grid) * a.cols * 2 * sizeof(float), &partial));
    const cudaError_t e = launch_pdl(
        kernel, dim3(static_cast<unsigned>(grid)), dim3(block), smem, ctx->stream, static_cast<const T*>(a.x),
        static_cast<const GT*>(a.gamma), static_cast<const T*>(a.dy), static_cast<T*>(a.dx),
        static_cast<float*>(partial), a.rows, static_cast<int>(a.cols), a.eps);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_layer_norm_bwd");
    QSML_TRY_STATUS(after_launch(ctx, "k_layer_norm_bwd"));
    return a.sums() ? finish(ctx, a, static_cast<float*>(partial), grid) : QSML_OK;
}

template <typename T, typename GT>
qsml_status_t launch_wide_bwd(Context* ctx, const Args& a) {
    Workspace ws(ctx);
    void *stats = nullptr, *partial = nullptr;
    // a chunk of rows for each CTA of the column kernel, about four CTAs an SM
    const int64_t tiles = (a.cols + 255) / 256;
    int64_t parts = (4 * ctx->num_sms + tiles - 1) / tiles;
    if (parts > a.rows) parts = a.rows;
    const int64_t chunk = (a.rows + parts - 1) / parts;
    parts = (a.rows + chunk - 1) / chunk;
    if (a.sums()) {
        QSML_TRY_STATUS(ws.get(static_cast<size_t>(a.rows) * sizeof(float2), &stats));
        QSML_TRY_STATUS(ws.get(static_cast<size_t>(parts) * a.cols * 2 * sizeof(float), &partial));
    }
    const int64_t grid = a.rows < 4 * ctx->num_sms ? a.rows : 4 * ctx->num_sms;
    cudaError_t e = launch_pdl(k_layer_norm_bwd_rows<T, GT>, dim3(static_cast<unsigned>(grid)), dim3(512), 0,
                               ctx->stream, static_cast<const T*>(a.x), static_cast<const GT*>(a.gamma),
                               static_cast<const T*>(a.dy), static_cast<T*>(a.dx), static_cast<float2*>(stats), a.rows,
                               a.cols, a.eps);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_layer_norm_bwd_rows");
    QSML_TRY_STATUS(after_launch(ctx, "k_layer_norm_bwd_rows"));
    if (!a.sums()) return QSML_OK;
    e = launch_pdl(k_layer_norm_bwd_cols<T>, dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(parts)),
                   dim3(256), 0, ctx->stream, static_cast<const T*>(a.x), static_cast<const T*>(a.dy),
                   static_cast<const float2*>(stats), static_cast<float*>(partial), a.rows, a.cols, chunk);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_layer_norm_bwd_cols");
    QSML_TRY_STATUS(after_launch(ctx, "k_layer_norm_bwd_cols"));
    return finish(ctx, a, static_cast<float*>(partial), parts);
}

// Columns by loads of PV elements: a warp a row while its lanes hold the row in
// 16 elements each, else a CTA with up to 16 elements a thread and 512 threads.
template <typename T, typename GT, int PV>
qsml_status_t pick(Context* ctx, const Args& a) {
    constexpr int MAXV = 16 / PV;
    const int64_t packs = a.cols / PV;
    if (packs <= 32) return launch_bwd<T, GT, PV, 1, true>(ctx, a, 32);
    if (packs <= 32 * MAXV) return launch_bwd<T, GT, PV, MAXV, true>(ctx, a, 32);
    if (packs <= 512 * MAXV) {
        const int th = static_cast<int>(((packs + MAXV - 1) / MAXV + 31) / 32 * 32);
        return launch_bwd<T, GT, PV, MAXV, false>(ctx, a, th);
    }
    return launch_wide_bwd<T, GT>(ctx, a);
}

template <typename T, typename GT>
qsml_status_t run_bwd(Context* ctx, const Args& a) {
    constexpr int PV = 16 / sizeof(T);
    if (a.cols % PV == 0 && aligned16(a.x) && aligned16(a.dy) && (!a.dx || aligned16(a.dx)))
        return pick<T, GT, PV>(ctx, a);
    return pick<T, GT, 1>(ctx, a);
}

}  // namespace
}  // namespace qsml

using namespace qsml;

extern "C" qsml_status_t qsml_layer_norm_backward(qsml_ctx* handle, const qsml_tdesc* x, const qsml_tdesc* gamma,
                                                  const qsml_tdesc* dy, float eps, const qsml_tdesc* dx,
                                                  const qsml_tdesc* dgamma, const qsml_tdesc* dbeta) {
    QSML_CTX(handle);
    QSML_TRY_STATUS(check_desc(C_, x, "x"));
    QSML_TRY_STATUS(check_desc(C_, gamma, "gamma"));
    QSML_TRY_STATUS(check_desc(C_, dy, "dy"));
    const qsml_tdesc* outs[3] = {dx, dgamma, dbeta};
    const char* names[3] = {"dx", "dgamma", "dbeta"};
    for (int i = 0; i < 3; ++i)
        if (outs[i]) QSML_TRY_STATUS(check_desc(C_, outs[i], names[i]));
    if (x->ndim < 1) return set_error(C_, QSML_E_SHAPE, "qsml_layer_norm_backward: x needs at least one dim");
    if (x->dtype != QSML_F32 && x->dtype != QSML_F16)
        return set_error(C_, QSML_E_DTYPE, "qsml_layer_norm_backward: x must be F32 or F16");
    if (dy->dtype != x->dtype || (dx && dx->dtype != x->dtype))
        return set_error(C_, QSML_E_DTYPE, "qsml_layer_norm_backward: dy and dx must have x's dtype");
    if (gamma->dtype != QSML_F32 && gamma->dtype != x->dtype)
        return set_error(C_, QSML_E_DTYPE, "qsml_layer_norm_backward: gamma must be F32 or x's dtype");
    for (int i = 1; i < 3; ++i)
        if (outs[i] && outs[i]->dtype != QSML_F32 && outs[i]->dtype != x->dtype)
            return set_error(C_, QSML_E_DTYPE, "qsml_layer_norm_backward: dgamma and dbeta must be F32 or x's dtype");
    if (!is_contiguous(x) || !is_contiguous(dy) || !is_contiguous(gamma))
        return set_error(C_, QSML_E_UNSUPPORTED, "qsml_layer_norm_backward: x, dy and gamma must be contiguous");
    const int64_t cols = x->shape[x->ndim - 1];
    const qsml_tdesc* like[2] = {dy, dx};
    for (const qsml_tdesc* t : like) {
        if (!t) continue;
        bool same = t->ndim == x->ndim;
        for (int d = 0; same && d < x->ndim; ++d) same = t->shape[d] == x->shape[d];
        if (!same) return set_error(C_, QSML_E_SHAPE, "qsml_layer_norm_backward: dy and dx must have x's shape");
    }
    if (numel(gamma) != cols) return set_error(C_, QSML_E_SHAPE, "qsml_layer_norm_backward: gamma must have the last dim's size");
    for (int i = 0; i < 3; ++i) {
        if (!outs[i]) continue;
        if (i > 0 && numel(outs[i]) != cols)
            return set_error(C_, QSML_E_SHAPE, "qsml_layer_norm_backward: dgamma and dbeta must have the last dim's size");
        if (!is_contiguous(outs[i]))
            return set_error(C_, QSML_E_UNSUPPORTED, "qsml_layer_norm_backward: outputs must be contiguous");
        bool meets = views_meet(outs[i], x) || views_meet(outs[i], dy) || views_meet(outs[i], gamma);
        for (int j = 0; j < i; ++j) meets = meets || (outs[j] && views_meet(outs[i], outs[j]));
        if (meets)
            return set_error(C_, QSML_E_INVALID, "qsml_layer_norm_backward: an output overlaps an input or another output");
    }
    if (cols == 0) return QSML_OK;
    const int64_t rows = numel(x) / cols;
    if (rows == 0) {  // sums over no rows
        for (int i = 1; i < 3; ++i)
            if (outs[i])
                QSML_TRY_STATUS(check_cuda(C_, cudaMemsetAsync(outs[i]->data, 0, cols * dtype_size(outs[i]->dtype), C_->stream),
                                           "qsml_layer_norm_backward zero"));
        return QSML_OK;
    }
    if (!dx && !dgamma && !dbeta) return QSML_OK;
    if (cols > INT32_MAX) return set_error(C_, QSML_E_UNSUPPORTED, "qsml_layer_norm_backward: rows of 2^31 elements or more");
    Args a;
    a.x = x->data;
    a.gamma = gamma->data;
    a.dy = dy->data;
    a.dx = dx ? dx->data : nullptr;
    if (dgamma) {
        a.sg.out = dgamma->data;
        a.sg.out_dtype = dgamma->dtype;
    }
    if (dbeta) {
        a.sb.out = dbeta->data;
        a.sb.out_dtype = dbeta->dtype;
    }
    a.rows = rows;
    a.cols = cols;
    a.eps = eps;
    if (x->dtype == QSML_F32) return run_bwd<float, float>(C_, a);
    if (gamma->dtype == QSML_F32) return run_bwd<__half, float>(C_, a);
    return run_bwd<__half, __half>(C_, a);
}
