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

// A CTA takes 8 columns (one 32-byte sector a row), its 64 groups of 8 lanes every
// 64th partial row, 8 rows in flight each; then a tree over the groups.  Bound by
// L2 latency: with 32 columns a CTA, 1184 rows of 1024 columns took 18 us.
constexpr int kFinishGroups = 64;

__global__ void __launch_bounds__(8 * kFinishGroups) k_column_finish(ColumnSum s0, ColumnSum s1, int64_t parts, int64_t cols) {
    pdl_begin();
    const ColumnSum s = blockIdx.y == 0 ? s0 : s1;
    __shared__ float acc[kFinishGroups][9];
    const int k = threadIdx.x & 7, group = threadIdx.x >> 3;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 8 + k;
    float a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = 0.0f;
    if (c < cols) {
        const float* p = s.partial + c;
        for (int64_t r = group; r < parts; r += 8 * kFinishGroups) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (r + i * kFinishGroups < parts) a[i] = __fadd_rn(a[i], p[(r + i * kFinishGroups) * cols]);
        }
    }
    acc[group][k] = __fadd_rn(__fadd_rn(__fadd_rn(a[0], a[1]), __fadd_rn(a[2], a[3])),
                              __fadd_rn(__fadd_rn(a[4], a[5]), __fadd_rn(a[6], a[7])));
    __syncthreads();
    // warp w < 8 owns column w: two of the 64 sums a lane
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    if (w >= 8) return;
    float v = __fadd_rn(acc[lane][w], acc[lane + 32][w]);
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, m));
    const int64_t oc = static_cast<int64_t>(blockIdx.x) * 8 + w;
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
    const dim3 grid(static_cast<unsigned>((cols + 7) / 8), n);
    const cudaError_t e = launch_pdl(k_column_finish, grid, dim3(8 * kFinishGroups), 0, ctx->stream, first, s1, parts, cols);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_column_finish");
    return after_launch(ctx, "k_column_finish");
}

}  // namespace qsml
