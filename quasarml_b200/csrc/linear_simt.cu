// The linear layers' products on the CUDA cores: any strides, sizes and
// alignment, one binary32 fma per k, k ascending.  128 x 64 outputs a CTA (twice
// that for a dual product), 4 rows x 8 columns a thread, k slices of 16 staged
// in shared memory with the next slice's loads in flight.  It serves
// QSML_MM_FP32_FFMA and products with nothing to sum.  Bound by the FFMA pipe on
// large products.
#include "linear.cuh"

namespace qsml {
namespace linear {
namespace {

constexpr int SM = 128, SN = 64, SK = 16;

template <typename T, bool DUAL>
__global__ void __launch_bounds__(256) k_linear_simt(const __grid_constant__ Problem p, int tiles_n) {
    pdl_begin();
    constexpr int NB = DUAL ? 2 : 1;
    __shared__ __align__(16) float As[SK][SM + 4];
    __shared__ __align__(16) float Bs[NB][SK][SN + 4];
    const int t = threadIdx.x, tx = t & 7, ty = t >> 3;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x / tiles_n) * SM;
    const int64_t col0 = static_cast<int64_t>(blockIdx.x % tiles_n) * SN;
    float acc[NB][4][8];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[b][i][j] = 0.0f;

    for (int s = 0; s < p.segments; ++s) {
        const Mat a = p.a[s];
        const bool a_k = a.cs == 1;  // neighbouring threads read neighbouring elements
        float ra[8], rb[NB][4];
        auto load = [&](int64_t k0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = t + i * 256;
                const int64_t m = row0 + (a_k ? e / SK : e % SM), k = k0 + (a_k ? e % SK : e / SM);
                ra[i] = m < p.M && k < p.K ? ld1(static_cast<const T*>(a.p) + m * a.rs + k * a.cs) : 0.0f;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const Mat w = p.b[DUAL ? b : s];
                const bool b_n = w.cs == 1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = t + i * 256;
                    const int64_t n = col0 + (b_n ? e % SN : e / SK), k = k0 + (b_n ? e / SN : e % SK);
                    rb[b][i] = n < p.N && k < p.K ? ld1(static_cast<const T*>(w.p) + k * w.rs + n * w.cs) : 0.0f;
                }
            }
        };
        if (p.K > 0) load(0);
        for (int64_t k0 = 0; k0 < p.K; k0 += SK) {
            __syncthreads();  // the slice before has been read
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = t + i * 256;
                As[a_k ? e % SK : e / SM][a_k ? e / SK : e % SM] = ra[i];
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const bool b_n = p.b[DUAL ? b : s].cs == 1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = t + i * 256;
                    Bs[b][b_n ? e / SN : e % SK][b_n ? e % SN : e / SK] = rb[b][i];
                }
            }
            __syncthreads();
            if (k0 + SK < p.K) load(k0 + SK);
            // only the k inside: no fma with padding
            const int kn = p.K - k0 < SK ? static_cast<int>(p.K - k0) : SK;
#pragma unroll 4
            for (int k = 0; k < kn; ++k) {
                const float4 av = *reinterpret_cast<const float4*>(&As[k][ty * 4]);
                const float am[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const float4 b0 = *reinterpret_cast<const float4*>(&Bs[b][k][tx * 8]);
                    const float4 b1 = *reinterpret_cast<const float4*>(&Bs[b][k][tx * 8 + 4]);
                    const float bn[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 8; ++j) acc[b][i][j] = __fmaf_rn(am[i], bn[j], acc[b][i][j]);
                }
            }
        }
        __syncthreads();
    }
    const int64_t col = col0 + tx * 8;
    if (col >= p.N) return;
    float bias[NB][8];
    bias8<T, DUAL>(p.e, col, bias);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = row0 + ty * 4 + i;
        if (row < p.M) finish8<T, DUAL>(p.e, row, col, bias, acc[0][i], acc[NB - 1][i]);
    }
}

}  // namespace

template <typename T> qsml_status_t run_simt(Context* ctx, const Problem& p) {
    const int64_t tm = (p.M + SM - 1) / SM, tn = (p.N + SN - 1) / SN;
    if (tm * tn > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "linear: too many output tiles");
    const cudaError_t e = launch_pdl(p.dual ? k_linear_simt<T, true> : k_linear_simt<T, false>,
                                     dim3(static_cast<unsigned>(tm * tn)), dim3(256), 0, ctx->stream, p,
                                     static_cast<int>(tn));
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_linear_simt");
    return after_launch(ctx, "k_linear_simt");
}

template qsml_status_t run_simt<float>(Context*, const Problem&);
template qsml_status_t run_simt<__half>(Context*, const Problem&);

}  // namespace linear
}  // namespace qsml
