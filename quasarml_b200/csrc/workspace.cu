// Workspace of one call and the joining of column sums (see workspace.cuh).
#include "workspace.cuh"

namespace qsml {

Workspace::~Workspace() {
    std::string err;
    for (int i = 0; i < n_; ++i) {
        if (captured_[i])
            cudaFreeAsync(ptr_[i], ctx_->stream);
        else
            ctx_->allocator->free(ptr_[i], &err);
    }
}

qsml_status_t Workspace::get(size_t bytes, void** ptr) {
    if (n_ == kMax) return set_error(ctx_, QSML_E_INVALID, "workspace: too many blocks");
    if (bytes == 0) bytes = 1;
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    QSML_TRY_STATUS(check_cuda(ctx_, cudaStreamIsCapturing(ctx_->stream, &cs), "workspace: capture status"));
    captured_[n_] = cs != cudaStreamCaptureStatusNone;
    if (captured_[n_]) {
        QSML_TRY_STATUS(check_cuda(ctx_, cudaMallocAsync(&ptr_[n_], bytes, ctx_->stream), "workspace of a captured call"));
    } else {
        std::string err;
        const qsml_status_t st = ctx_->allocator->alloc(bytes, &ptr_[n_], &err);
        if (st != QSML_OK) return set_error(ctx_, st, err);
    }
    *ptr = ptr_[n_++];
    return QSML_OK;
}

namespace {

// A CTA takes 32 columns; its 32 warps take every 32nd partial row, each lane
// one column (128-byte rows), then warp 0 adds the 32 warps' sums in order.
// Bound by L2 latency: a few thousand rows of 32 columns per CTA at most.
__global__ void __launch_bounds__(1024) k_column_finish(ColumnSum s0, ColumnSum s1, int64_t parts, int64_t cols) {
    pdl_begin();
    const ColumnSum s = blockIdx.y == 0 ? s0 : s1;
    __shared__ float acc[32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float a0 = 0.0f, a1 = 0.0f, a2 = 0.0f, a3 = 0.0f;
    if (c < cols) {
        const float* p = s.partial + c;
        int64_t r = w;
        for (; r + 96 < parts; r += 128) {
            a0 = __fadd_rn(a0, p[r * cols]);
            a1 = __fadd_rn(a1, p[(r + 32) * cols]);
            a2 = __fadd_rn(a2, p[(r + 64) * cols]);
            a3 = __fadd_rn(a3, p[(r + 96) * cols]);
        }
        for (; r < parts; r += 32) a0 = __fadd_rn(a0, p[r * cols]);
    }
    acc[w][lane] = __fadd_rn(__fadd_rn(a0, a1), __fadd_rn(a2, a3));
    __syncthreads();
    // warp w now owns column w: its lanes hold the 32 partial sums
    float v = acc[lane][w];
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, m));
    const int64_t oc = static_cast<int64_t>(blockIdx.x) * 32 + w;
    if (lane == 0 && oc < cols) {
        if (s.out_dtype == QSML_F16)
            static_cast<__half*>(s.out)[oc] = __float2half_rn(v);
        else
            static_cast<float*>(s.out)[oc] = v;
    }
}

}  // namespace

qsml_status_t finish_column_sums(Context* ctx, const ColumnSum& s0, const ColumnSum& s1, int64_t parts, int64_t cols) {
    const ColumnSum first = s0.out ? s0 : s1;
    const unsigned n = (s0.out ? 1u : 0u) + (s1.out ? 1u : 0u);
    if (n == 0 || cols == 0) return QSML_OK;
    const dim3 grid(static_cast<unsigned>((cols + 31) / 32), n);
    const cudaError_t e = launch_pdl(k_column_finish, grid, dim3(1024), 0, ctx->stream, first, s1, parts, cols);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_column_finish");
    return after_launch(ctx, "k_column_finish");
}

}  // namespace qsml
