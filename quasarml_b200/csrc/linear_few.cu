// The linear layers of a few rows in binary32 (a token, a handful of them): the
// weight is read once as it lies, with binary32 fma on the CUDA cores.  The tensor
// cores' three parts would move it four times (16 bytes an element for 4: one row
// through 4096 x 4096 took 50 us).  Bound by HBM up to 8 rows, by the fma pipe
// near 16.
//
// A CTA takes COLS columns; a cluster of up to 8 shares the sum over k, and their
// binary32 sums meet in distributed shared memory, added in rank order.
//   N contiguous: 128 columns, 4 a lane; the 8 warps take every eighth k each;
//   K contiguous: 32 columns, 4 a warp; the lanes take k.
#include "linear.cuh"

namespace qsml {
namespace linear {
namespace {

constexpr int KC = 256;       // k of x staged in shared memory at a time
constexpr int THREADS = 256;

__device__ __forceinline__ void ld4(const float* p, float (&v)[4]) {
    const float4 f = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
}

// M rows (a template bound MR, rows past p.M are zero).  VEC: 16-byte loads of the
// weight.  KMAJOR: k contiguous in the weight.
template <int MR, bool DUAL, bool KMAJOR, bool VEC>
__global__ void __launch_bounds__(THREADS) k_linear_few(const __grid_constant__ Problem p, int splits) {
    pdl_begin();
    constexpr int NB = DUAL ? 2 : 1;
    constexpr int COLS = KMAJOR ? 32 : 128;
    extern __shared__ __align__(16) float few_smem[];
    float* xs = few_smem;                              // N contiguous: [KC][MR], else [MR][KC]
    float* part = few_smem + KC * MR;                  // [NB][8 warps or 1][MR][COLS]
    constexpr int COPIES = KMAJOR ? 1 : 8;
    const int t = threadIdx.x, lane = t & 31, w = t >> 5;
    const int tile = static_cast<int>(blockIdx.x) / splits, rank = static_cast<int>(blockIdx.x) % splits;
    const int64_t n0 = static_cast<int64_t>(tile) * COLS;
    const int64_t chunks = (p.K + KC - 1) / KC, total = chunks * p.segments;
    const int64_t c0 = total * rank / splits, c1 = total * (rank + 1) / splits;
    float acc[NB][MR][4];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[b][m][j] = 0.0f;

    for (int64_t c = c0; c < c1; ++c) {
        const int s = static_cast<int>(c / chunks);
        const int64_t k0 = (c - s * chunks) * KC;
        const int kn = p.K - k0 < KC ? static_cast<int>(p.K - k0) : KC;
        const Mat a = p.a[s];
        __syncthreads();
        for (int i = t; i < KC * MR; i += THREADS) {
            const int k = i % KC, m = i / KC;
            const float v = k < kn && m < p.M ? static_cast<const float*>(a.p)[m * a.rs + (k0 + k) * a.cs] : 0.0f;
            xs[KMAJOR ? m * KC + k : k * MR + m] = v;
        }
        __syncthreads();
        if constexpr (!KMAJOR) {
            // lane's columns: 4 together, or every 32nd
            constexpr int U = MR >= 8 ? 4 : 8;  // rows of the weight in flight
            for (int i = w; i < kn; i += 8 * U) {
                float v[NB][U][4];
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const Mat wt = p.b[DUAL ? b : s];
                        const float* row = static_cast<const float*>(wt.p) + (k0 + i + 8 * u) * wt.rs + n0;
                        const bool in = i + 8 * u < kn;
                        if constexpr (VEC) {
                            if (in && n0 + lane * 4 < p.N) {
                                ld4(row + lane * 4, v[b][u]);
                            } else {
#pragma unroll
                                for (int j = 0; j < 4; ++j) v[b][u][j] = 0.0f;
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                v[b][u][j] = in && n0 + j * 32 + lane < p.N ? __ldg(row + j * 32 + lane) : 0.0f;
                        }
                    }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (i + 8 * u >= kn) break;  // no fma with padding
#pragma unroll
                    for (int m = 0; m < MR; ++m) {
                        const float x = xs[(i + 8 * u) * MR + m];
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int j = 0; j < 4; ++j) acc[b][m][j] = __fmaf_rn(x, v[b][u][j], acc[b][m][j]);
                    }
                }
            }
        } else {
            constexpr int STEP = VEC ? 128 : 32, E = VEC ? 4 : 1;  // k a round, k a lane of it
            for (int i = 0; i < kn; i += STEP) {
                const int k = i + lane * E;
                float v[NB][4][E];
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const Mat wt = p.b[DUAL ? b : s];
                        const int64_t n = n0 + w * 4 + j;
                        const float* q = static_cast<const float*>(wt.p) + n * wt.cs + k0 + k;
                        if constexpr (VEC) {
                            if (n < p.N && k < kn) {
                                ld4(q, v[b][j]);
                            } else {
#pragma unroll
                                for (int e = 0; e < E; ++e) v[b][j][e] = 0.0f;
                            }
                        } else {
                            v[b][j][0] = n < p.N && k < kn ? __ldg(q) : 0.0f;
                        }
                    }
                if (k < kn) {
#pragma unroll
                    for (int m = 0; m < MR; ++m)
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const float x = xs[m * KC + k + e];
#pragma unroll
                            for (int b = 0; b < NB; ++b)
#pragma unroll
                                for (int j = 0; j < 4; ++j) acc[b][m][j] = __fmaf_rn(x, v[b][j][e], acc[b][m][j]);
                        }
                }
            }
        }
    }
    // this CTA's sums: [b][copy][m][column]
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (KMAJOR) {
                    float v = acc[b][m][j];
#pragma unroll
                    for (int x = 16; x >= 1; x >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, x));
                    if (lane == 0) part[(b * MR + m) * COLS + w * 4 + j] = v;
                } else {
                    part[((b * COPIES + w) * MR + m) * COLS + (VEC ? lane * 4 + j : j * 32 + lane)] = acc[b][m][j];
                }
            }
    __syncthreads();
    if constexpr (!KMAJOR) {
        for (int i = t; i < NB * MR * COLS; i += THREADS) {
            const int b = i / (MR * COLS), r = i % (MR * COLS);
            float* q = part + b * COPIES * MR * COLS + r;
            float v = q[0];
#pragma unroll
            for (int k = 1; k < 8; ++k) v = __fadd_rn(v, q[k * MR * COLS]);
            q[0] = v;
        }
        __syncthreads();
    }
    if (splits > 1)
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(part));
    const int64_t M = p.M < MR ? p.M : MR;
    for (int i = rank * THREADS + t; i < M * (COLS / 8); i += splits * THREADS) {
        const int m = i / (COLS / 8), c = i % (COLS / 8) * 8;
        if (n0 + c >= p.N) continue;
        float z[2][8];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint32_t at = base + ((b * COPIES * MR + m) * COLS + c) * 4;
#pragma unroll
            for (int j = 0; j < 8; ++j) z[b][j] = 0.0f;
            for (int s = 0; s < splits; ++s) {
                uint32_t from;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(at), "r"(s));
                float f[8];
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(f[4 * h]), "=f"(f[4 * h + 1]), "=f"(f[4 * h + 2]), "=f"(f[4 * h + 3])
                                 : "r"(from + 16 * h)
                                 : "memory");
#pragma unroll
                for (int j = 0; j < 8; ++j) z[b][j] = s ? __fadd_rn(z[b][j], f[j]) : f[j];
            }
        }
        float bias[NB][8];
        bias8<float, DUAL>(p.e, n0 + c, bias);
        finish8<float, DUAL>(p.e, m, n0 + c, bias, z[0], z[1]);
    }
    if (splits > 1)  // no CTA leaves while another reads its sums
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

template <int MR, bool DUAL, bool KMAJOR, bool VEC> qsml_status_t launch(Context* ctx, const Problem& p) {
    auto kernel = k_linear_few<MR, DUAL, KMAJOR, VEC>;
    constexpr int COLS = KMAJOR ? 32 : 128;
    constexpr size_t smem = sizeof(float) * (KC * MR + (DUAL ? 2 : 1) * (KMAJOR ? 1 : 8) * MR * COLS);
    {
        static std::mutex mu;
        static uint64_t done = 0;
        std::lock_guard<std::mutex> lk(mu);
        const uint64_t bit = uint64_t(1) << (ctx->device & 63);
        if (smem > 40 * 1024 && !(done & bit)) {
            QSML_TRY_STATUS(check_cuda(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                                 static_cast<int>(smem)),
                                       "linear: shared-memory attribute"));
            done |= bit;
        }
    }
    const int64_t tiles = (p.N + COLS - 1) / COLS, chunks = (p.K + KC - 1) / KC * p.segments;
    if (tiles * 8 > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "linear: too many output tiles");
    // about two CTAs a SM
    int64_t splits = (2 * ctx->num_sms) / tiles;
    splits = splits < 1 ? 1 : splits > 8 ? 8 : splits;
    if (splits > chunks) splits = chunks;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(splits);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * splits));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cfg.attrs = attr;
    cfg.numAttrs = splits > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p, static_cast<int>(splits));
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_linear_few");
    return after_launch(ctx, "k_linear_few");
}

template <bool DUAL, bool KMAJOR, bool VEC> qsml_status_t by_rows(Context* ctx, const Problem& p) {
    if (p.M <= 1) return launch<1, DUAL, KMAJOR, VEC>(ctx, p);
    if (p.M <= 4) return launch<4, DUAL, KMAJOR, VEC>(ctx, p);
    if (p.M <= 8) return launch<8, DUAL, KMAJOR, VEC>(ctx, p);
    if constexpr (!DUAL) return launch<16, DUAL, KMAJOR, VEC>(ctx, p);
    return QSML_E_UNSUPPORTED;
}

}  // namespace

bool few_rows(const Problem& p) {
    if (p.M > (p.dual ? 8 : 16) || p.K == 0) return false;
    const int nb = p.dual ? 2 : p.segments;
    bool n_major = true, k_major = true;
    for (int i = 0; i < p.segments; ++i)
        if (p.a[i].plane) return false;  // split for the tensor cores
    for (int i = 0; i < nb; ++i) {
        if (p.b[i].plane) return false;
        n_major = n_major && p.b[i].cs == 1;
        k_major = k_major && p.b[i].rs == 1;
    }
    return n_major || k_major;
}

qsml_status_t run_few(Context* ctx, const Problem& p) {
    const int nb = p.dual ? 2 : p.segments;
    bool n_major = true, vec = true;
    for (int i = 0; i < nb; ++i) n_major = n_major && p.b[i].cs == 1;
    for (int i = 0; i < nb; ++i)
        vec = vec && aligned16(p.b[i].p) && (n_major ? p.b[i].rs % 4 == 0 && p.N % 4 == 0 : p.b[i].cs % 4 == 0 && p.K % 4 == 0);
    if (n_major) {
        if (p.dual) return vec ? by_rows<true, false, true>(ctx, p) : by_rows<true, false, false>(ctx, p);
        return vec ? by_rows<false, false, true>(ctx, p) : by_rows<false, false, false>(ctx, p);
    }
    if (p.dual) return vec ? by_rows<true, true, true>(ctx, p) : by_rows<true, true, false>(ctx, p);
    return vec ? by_rows<false, true, true>(ctx, p) : by_rows<false, true, false>(ctx, p);
}

}  // namespace linear
}  // namespace qsml
