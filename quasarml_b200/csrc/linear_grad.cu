// Gradients of the linear layers with respect to their products, and the
// biases' gradients: one pass over dy and what the forward pass kept.
//   LINEAR: dz = dy act'(pre)            db = column sums of dz
//   DUAL:   dg = dy u act'(g), du = dy act(g), and the column sums of both
// dz goes to a workspace that the two products of the backward pass read (in the parts
// that the tensor cores take, see GradArgs); the sums are taken before it is rounded.
//
// binary16's dz is stored times a power of two s, which the products' epilogue undoes:
// dy u can be far beyond binary16 where dx and dw are not, and a small dz is held in few
// bits where a sum of many is an ordinary number.  s is one number for the whole of dz
// (dg and du), since dx sums over its columns and dw over its rows.  It is 2^8 if
// the largest finite |dz| turns out to be in [1, 255], which is known behind a barrier of
// the grid or, where few CTAs do, of a cluster (7 us of the 164 of a backward pass of
// 16384 x 1024 x 2048; of small ones, back to back, 4 with the grid's cooperative launch and
// 2 with a cluster).  If not, the CTAs go over their inputs again, with the s that
// brings the largest into [2^14, 2^15) (37 us more there).  Either way an element keeps
// binary16's 11 bits, or is off by 2^-25 of the scaled numbers' unit, 2^-33 of the largest.
// Bound by HBM: LINEAR reads 2 and writes 1 element, DUAL reads 3 and writes 2 (binary16:
// 16384 x 2048 with gelu 45 us, 4.5 TB/s; DUAL 8192 x 5632 79 us, 5.8 TB/s).
#include <cfloat>

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

// The largest of the block's values, in every thread.
__device__ __forceinline__ float block_max(float v) {
    __shared__ float by_warp[8];
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, m));
    if ((threadIdx.x & 31) == 0) by_warp[threadIdx.x >> 5] = v;
    __syncthreads();
    v = by_warp[0];
#pragma unroll
    for (int k = 1; k < 8; ++k) v = fmaxf(v, by_warp[k]);
    __syncthreads();
    return v;
}

// The largest finite magnitude among eight values (0 if there is none).
__device__ __forceinline__ float largest(const P2 (&d)[4]) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 e = unpack(d[j]);
        m = fmaxf(m, fmaxf(fabsf(e.x), fabsf(e.y)));  // passes over NaN
    }
    if (m <= FLT_MAX) return m;
    m = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 e = unpack(d[j]);
        if (fabsf(e.x) <= FLT_MAX) m = fmaxf(m, fabsf(e.x));
        if (fabsf(e.y) <= FLT_MAX) m = fmaxf(m, fabsf(e.y));
    }
    return m;
}

// The block's writes are seen by all blocks that pass, once all of the grid have come and *arrived
// is `all`.  False if they do not come within the default limit (the device holds the whole grid,
// so only where something is wrong).
__device__ __forceinline__ bool grid_barrier(unsigned* arrived, unsigned all) {
    int here = 1;
    if (threadIdx.x == 0) {
        asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(arrived) : "memory");
        const long long t0 = clock64();
        for (unsigned n = 0;;) {
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(arrived) : "memory");
            if (static_cast<int>(n - all) >= 0) break;
            if (clock64() - t0 > kDefaultWaitCycles) {
                here = 0;
                break;
            }
        }
    }
    return __syncthreads_and(here) != 0;
}

constexpr int kDzExponent = 8;
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// An item is 256 columns (8 a lane) by `chunk` rows, a CTA's 8 warps taking every 8th row;
// items go round the grid, columns first.  A thread keeps its columns and sums them in
// registers; the warps' sums are added in warp order in shared memory.
// SCALED: dz times a power of two (above); the grid is cooperative, or one cluster (no `arrived`).
template <typename T, bool DUAL, int ACT, bool SCALED>
__global__ void __launch_bounds__(256, DUAL ? 2 : 3)
    k_linear_dz(const __grid_constant__ GradArgs a, int64_t chunk, int tiles, int items, bool vec) {
    pdl_begin();
    constexpr int NO = DUAL ? 2 : 1;
    __shared__ float fold[NO][8][256 + 8];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    float scale = power_of_two(kDzExponent), most = 0.0f;
    bool again = false;  // the second time: neither sums nor the largest
    for (int item = blockIdx.x;; item += gridDim.x) {
        if (item >= items) {
            if (!SCALED || again) return;
            most = block_max(most);
            if (threadIdx.x == 0) a.most[blockIdx.x] = most;
            bool met = true;
            if (a.arrived) met = grid_barrier(a.arrived, a.all);
            else asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
            if (!met) {
                if (threadIdx.x == 0) atomicExch(a.status, QSML_E_TIMEOUT);
                return;
            }
            most = 0.0f;
            for (unsigned i = threadIdx.x; i < gridDim.x; i += 256) most = fmaxf(most, a.most[i]);
            most = block_max(most);
            const bool fits = most == 0.0f || (most >= 1.0f && most <= 255.0f);
            const int e = fits ? kDzExponent : min(14 - ilogbf(most), 100);
            if (blockIdx.x == 0 && threadIdx.x == 0) *a.unscale = power_of_two(-e);
            if (fits) return;
            scale = power_of_two(e);
            again = true;
            item = blockIdx.x;
        }
        const int64_t col = static_cast<int64_t>(item % tiles) * 256 + lane * 8;
        const int n = a.N - col < 8 ? static_cast<int>(a.N - col) : 8;  // may be <= 0
        const int64_t r0 = item / tiles * chunk, r1 = r0 + chunk < a.M ? r0 + chunk : a.M;
        const bool sums = a.partial && !again;
        P2 sum[NO][4];
#pragma unroll
        for (int o = 0; o < NO; ++o)
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[o][j].v = 0;
        if (n > 0) {
            // AHEAD rows in flight under the one at hand: as many as leave two CTAs a SM, three
            // LINEAR ones of binary16 (DUAL binary16 8192 x 5632, not scaled: 88, 79, 76 us with 1, 2, 3;
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
                    if (sums) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) sum[o][j] = add2(sum[o][j], d[o][j]);
                    }
                    if (a.dz[o]) {
                        float f[8];
                        if constexpr (SCALED) {
                            if (!again) most = fmaxf(most, largest(d[o]));
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 e = unpack(SCALED ? mul2(d[o][j], both(scale)) : d[o][j]);
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
        if (!sums) continue;
#pragma unroll
        for (int o = 0; o < NO; ++o)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 e = unpack(sum[o][j]);
                fold[o][w][lane * 8 + 2 * j] = e.x;
                fold[o][w][lane * 8 + 2 * j + 1] = e.y;
            }
        __syncthreads();
        const int64_t c = static_cast<int64_t>(item % tiles) * 256 + threadIdx.x;
        if (c < a.N) {
#pragma unroll
            for (int o = 0; o < NO; ++o) {
                float s = fold[o][0][threadIdx.x];
                for (int k = 1; k < 8; ++k) s = __fadd_rn(s, fold[o][k][threadIdx.x]);
                a.partial[(static_cast<int64_t>(o) * (items / tiles) + item / tiles) * a.N + c] = s;
            }
        }
        __syncthreads();  // the sums have been read
    }
}

// CTAs of a cooperative launch that the device holds at once, once a device and kernel.
template <typename T, bool DUAL, int ACT> qsml_status_t resident(Context* ctx, int64_t* ctas) {
    static std::mutex mu;
    static int known[64] = {};
    std::lock_guard<std::mutex> lk(mu);
    int& n = known[ctx->device & 63];
    if (n == 0) {
        int per_sm = 0;
        QSML_TRY_STATUS(check_cuda(ctx, cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k_linear_dz<T, DUAL, ACT, true>,
                                                                                      256, 0),
                                   "linear: occupancy"));
        if (per_sm < 1) return set_error(ctx, QSML_E_CUDA, "linear: k_linear_dz does not fit a SM");
        n = per_sm * ctx->num_sms;
    }
    *ctas = n;
    return QSML_OK;
}

constexpr int64_t MAX_CLUSTER = 8;  // portable

template <typename T, bool DUAL, int ACT> qsml_status_t launch_act(Context* ctx, const GradArgs& given) {
    GradArgs a = given;
    const int64_t tiles = (a.N + 255) / 256;
    // binary32's parts have its range, and binary16's dy without an activation is dz itself
    constexpr bool CAN_SCALE = sizeof(T) == 2 && (DUAL || ACT != QSML_ACT_NONE);
    const bool scaled = CAN_SCALE && a.unscale;
    // about eight items an SM, at least 2 rows a warp (8 left most SMs without a CTA at
    // 515 x 1366: 23 us); as many as the device holds where the grid is cooperative
    // (16384 x 2048, 440 items: three a CTA took 3 us more)
    int64_t held = 0, parts = (8 * ctx->num_sms + tiles - 1) / tiles;
    const int64_t most = (a.M + 15) / 16;
    // few items: one cluster, whose barrier needs no cooperative launch and none of its 2 us
    // (64 x 256 x 1024, 16 items, the whole pass: 15.5 us for 17.0; 32 items: 17.5 for 17.0)
    const bool cluster = scaled && tiles * most <= 16;
    if constexpr (CAN_SCALE) {
        if (cluster) {
            held = MAX_CLUSTER;
        } else if (scaled) {
            QSML_TRY_STATUS((resident<T, DUAL, ACT>(ctx, &held)));
        }
        if (scaled) parts = std::max<int64_t>(1, held / tiles);
    }
    if (parts > most) parts = most;
    const int64_t chunk = (a.M + parts - 1) / parts;
    parts = (a.M + chunk - 1) / chunk;
    const int64_t items = tiles * parts, grid = scaled && items > held ? held : items;
    Workspace ws(ctx);
    const bool sums = a.db[0].out || a.db[1].out;
    const size_t partial = sums ? static_cast<size_t>(DUAL ? 2 : 1) * parts * a.N : 0;
    void* memory = nullptr;
    const size_t floats = partial + (scaled ? grid + 1 : 0);  // 1: a captured cooperative call's barrier
    if (floats) QSML_TRY_STATUS(ws.get(floats * sizeof(float), &memory));
    if (sums) a.partial = static_cast<float*>(memory);
    if (scaled) {
        a.most = static_cast<float*>(memory) + partial;
        a.status = ctx->status;
        // The context's count of arrivals goes on from call to call, which are in stream order; a
        // captured call may be replayed beside them and counts on its own, from 0.
        if (!cluster && ws.captured()) {
            a.arrived = reinterpret_cast<unsigned*>(a.most + grid);
            a.all = static_cast<unsigned>(grid);
            QSML_TRY_STATUS(check_cuda(ctx, cudaMemsetAsync(a.arrived, 0, sizeof(unsigned), ctx->stream), "linear: barrier"));
        } else if (!cluster) {
            a.arrived = reinterpret_cast<unsigned*>(ctx->status + 4);
            a.all = ctx->arrivals + static_cast<unsigned>(grid);
        }
    }
    bool vec = a.N % 8 == 0 && a.dy_ld % 8 == 0 && aligned16(a.dy);
    for (int i = 0; i < 2; ++i) vec = vec && (!a.pre[i] || aligned16(a.pre[i]));
    // A grid with a barrier has to be on the device whole, whatever else runs there: a cooperative
    // launch, which does not begin before the kernel ahead of it has ended.
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = a.arrived ? cudaLaunchAttributeCooperative : cudaLaunchAttributeProgrammaticStreamSerialization;
    if (a.arrived) attr[0].val.cooperative = 1;
    else attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(grid);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(256);
    cfg.stream = ctx->stream;
    cfg.attrs = attr;
    cfg.numAttrs = cluster && grid > 1 ? 2 : 1;
    auto kernel = k_linear_dz<T, DUAL, ACT, false>;
    if constexpr (CAN_SCALE)
        if (scaled) kernel = k_linear_dz<T, DUAL, ACT, true>;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, chunk, static_cast<int>(tiles), static_cast<int>(items), vec);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_linear_dz");
    if (a.arrived && !ws.captured()) ctx->arrivals = a.all;
    QSML_TRY_STATUS(after_launch(ctx, "k_linear_dz"));
    if (!sums) return QSML_OK;
    ColumnSum s0 = a.db[0], s1 = a.db[1];
    s0.partial = a.partial;
    s1.partial = a.partial + parts * a.N;
    return finish_column_sums(ctx, s0, s1, parts, a.N);
}

template <typename T, bool DUAL> qsml_status_t launch(Context* ctx, const GradArgs& a) {
    switch (a.act) {
        case QSML_ACT_RELU: return launch_act<T, DUAL, QSML_ACT_RELU>(ctx, a);
        case QSML_ACT_GELU: return launch_act<T, DUAL, QSML_ACT_GELU>(ctx, a);
        case QSML_ACT_SILU: return launch_act<T, DUAL, QSML_ACT_SILU>(ctx, a);
        case QSML_ACT_SIGMOID: return launch_act<T, DUAL, QSML_ACT_SIGMOID>(ctx, a);
    }
    return launch_act<T, DUAL, QSML_ACT_NONE>(ctx, a);
}

}  // namespace

template <typename T> qsml_status_t run_grad(Context* ctx, const GradArgs& a, bool dual) {
    return dual ? launch<T, true>(ctx, a) : launch<T, false>(ctx, a);
}
template qsml_status_t run_grad<float>(Context*, const GradArgs&, bool);
template qsml_status_t run_grad<__half>(Context*, const GradArgs&, bool);

}  // namespace linear
}  // namespace qsml
