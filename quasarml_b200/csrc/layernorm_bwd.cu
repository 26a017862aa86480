// Backward pass of the layer norm over the last dim.  With
//   xh = (x - mean) rstd,  h = dy gamma,
//   c1 = mean_c(h),        c2 = mean_c(h xh)          (means along the row)
// the gradients are
//   dx = rstd (h - c1 - xh c2),   dgamma_c = sum_r dy xh,   dbeta_c = sum_r dy.
// The forward pass keeps nothing for it: mean and rstd are computed again from
// the row, which has to be read for xh anyway.  The reference has no layer
// norm and no gradients.
//
// k_layer_norm_bwd: a CTA holds a row of x and dy in registers, so both are read
// once and dx is written once (3 elements of traffic, the floor).  Rows of whole
// 16-byte groups come through a ring of shared-memory slots filled by bulk copies
// (bounded waits), other rows through registers one row ahead.  Row sums take two
// steps: the row sum, then together the squared deviations, sum(h) and
// sum(h (x - mean)), all about the mean, so nothing is lost by cancellation.  A
// thread keeps its columns for every row it meets and so sums dgamma and dbeta in
// registers (binary32); the CTAs' sums are joined by k_column_finish in a fixed
// order.  Arithmetic is in packed pairs (fma.rn.f32x2 and the like, each lane
// rounded as the scalar instruction): the kernel was bound by instructions, 32 an
// element, before it was by HBM.
// k_layer_norm_bwd_groups: rows narrower than a CTA's, 4 to 32 lanes a row.
// k_layer_norm_bwd_rows + k_layer_norm_bwd_cols: rows too wide for the registers to
// hold the columns' sums as well (8192 columns, 6144 off 16 bytes), in two kernels
// (5 elements of traffic and the row statistics; 4096 x 16384 binary16: 154 us).
#include "packed.cuh"
#include "row_pipe.cuh"
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

// Sums of N values over the CTA, every thread ending with the same bits.  `slot`
// (N x 32 floats) is not written again before every thread has read it: callers
// alternate two.
template <int N> __device__ __forceinline__ void row_sums(float (&v)[N], float* slot) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = warp_add(v[i]);
        if (lane == 0) slot[i * 32 + w] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_add(lane < nw ? slot[i * 32 + lane] : 0.0f);
}

// A thread's columns: NV groups of PV elements, group i at column
// (t + i * th) * PV of the row, as E / 2 pairs.
template <typename T, int PV, int NV> struct Cols {
    static constexpr int E = PV * NV, H = E / 2;
    using V = Vec<T, PV>;
    V v[NV];
    __device__ P2 pair(int j) const {  // elements 2 j and 2 j + 1
        if constexpr (sizeof(T) == 2 && PV >= 2) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[2 * j / PV].v[2 * j % PV]));
            return pack(f.x, f.y);
        } else {
            return pack(to_f(v[2 * j / PV].v[2 * j % PV]), to_f(v[(2 * j + 1) / PV].v[(2 * j + 1) % PV]));
        }
    }
    __device__ void set(int j, P2 p) {
        const float2 f = unpack(p);
        if constexpr (sizeof(T) == 2 && PV >= 2) {
            *reinterpret_cast<__half2*>(&v[2 * j / PV].v[2 * j % PV]) = __floats2half2_rn(f.x, f.y);
        } else {
            from_f(f.x, v[2 * j / PV].v[2 * j % PV]);
            from_f(f.y, v[(2 * j + 1) / PV].v[(2 * j + 1) % PV]);
        }
    }
};

// What a thread keeps of its columns over the rows, and the arithmetic of a row
// between the sums.  Columns past the row's end (not FULL) have x and dy 0; only
// their deviations need a mask.  With 32 elements a thread (WIDE) the registers
// go to the sums and the deviations: dy stays as it was loaded and gamma is read
// from shared memory, group p's quad k as float4 k * packs + p.
template <typename T, int PV, int NV, bool FULL> struct RowWork {
    using C = Cols<T, PV, NV>;
    static constexpr int H = C::H;
    static constexpr bool WIDE = C::E > 16;
    P2 g[WIDE ? 1 : H], sg[H], sb[H];
    P2 d[H], y[WIDE ? 1 : H];
    C raw;
    const float4* sgam;
    int t, th, packs;

    __device__ bool in(int i) const { return FULL || t + i * th < packs; }
    template <typename GT> __device__ void begin(const GT* gamma, float4* shared, int t_, int th_, int packs_) {
        t = t_;
        th = th_;
        packs = packs_;
        sgam = shared;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float f[PV];
#pragma unroll
            for (int e = 0; e < PV; ++e) f[e] = in(i) ? to_f(gamma[(t + i * th) * PV + e]) : 0.0f;
            if constexpr (WIDE) {
                if (in(i))
#pragma unroll
                    for (int k = 0; k < PV / 4; ++k)
                        shared[k * packs + t + i * th] = make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
            } else {
#pragma unroll
                for (int e = 0; e < PV; ++e) {
                    const int k = i * PV + e;
                    const float2 u = unpack(g[k / 2]);
                    g[k / 2] = k % 2 ? pack(u.x, f[e]) : pack(f[e], 0.0f);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < H; ++j) sg[j].v = sb[j].v = 0;
    }
    __device__ P2 dy(int j) const {
        if constexpr (WIDE) return raw.pair(j);
        else return y[j];
    }
    // gamma of pairs 2 q and 2 q + 1
    __device__ void gam(int q, P2 (&o)[2]) const {
        if constexpr (WIDE) {
            const int i = q / (PV / 4);
            const float4 f = sgam[q % (PV / 4) * packs + (in(i) ? t + i * th : 0)];
            o[0] = pack(f.x, f.y);
            o[1] = pack(f.z, f.w);
        } else {
            o[0] = g[2 * q];
            o[1] = g[2 * q + 1];
        }
    }
    // the row's values; their sum
    __device__ float take(const C& x, const C& dyv) {
        P2 s;
        s.v = 0;
        if constexpr (WIDE) raw = dyv;
#pragma unroll
        for (int j = 0; j < H; ++j) {
            d[j] = x.pair(j);
            if constexpr (!WIDE) y[j] = dyv.pair(j);
            s = add2(s, d[j]);
        }
        return sum2(s);
    }
    // x - mean; sums of its square, of h = dy gamma and of h (x - mean)
    __device__ void deviations(float mean, float (&s3)[3]) {
        const P2 m = pack(-mean, -mean);
        P2 q, a, b;
        q.v = a.v = b.v = 0;
#pragma unroll
        for (int k = 0; k < H / 2; ++k) {
            P2 gg[2];
            gam(k, gg);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int j = 2 * k + u;
                d[j] = add2(d[j], m);
                if (!FULL) {
                    const float2 f = unpack(d[j]);
                    d[j] = pack(in(2 * j / PV) ? f.x : 0.0f, in((2 * j + 1) / PV) ? f.y : 0.0f);
                }
                const P2 h = mul2(dy(j), gg[u]);
                q = fma2(d[j], d[j], q);
                a = add2(a, h);
                b = fma2(h, d[j], b);
            }
        }
        s3[0] = sum2(q);
        s3[1] = sum2(a);
        s3[2] = sum2(b);
    }
    // dx = rstd h - (rstd c1 + (x - mean) rstd^2 c2),  c2 = mean(h (x - mean)) rstd
    __device__ void outputs(const float (&s3)[3], float inv_n, float eps, C& out) {
        const float rstd = rsqrtf(__fmaf_rn(s3[0], inv_n, eps));
        const float a = __fmul_rn(__fmul_rn(s3[1], inv_n), -rstd);
        const float b = __fmul_rn(__fmul_rn(__fmul_rn(s3[2], inv_n), rstd), -__fmul_rn(rstd, rstd));
        const P2 r2 = pack(rstd, rstd), a2 = pack(a, a), b2 = pack(b, b);
#pragma unroll
        for (int k = 0; k < H / 2; ++k) {
            P2 gg[2];
            gam(k, gg);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int j = 2 * k + u;
                const P2 v = dy(j), h = mul2(v, gg[u]);
                out.set(j, fma2(h, r2, fma2(d[j], b2, a2)));
                sg[j] = fma2(v, mul2(d[j], r2), sg[j]);
                sb[j] = add2(sb[j], v);
            }
        }
    }
};

// Three values' sums over a warp, six exchanges instead of fifteen: two values
// change places by half warps, then by quarters, so that a lane goes on with one
// of them.  Lanes 0-7 end with v[0]'s sum, 8-15 with v[1]'s, 16-23 with v[2]'s.
__device__ __forceinline__ float warp_sum3(const float (&v)[3]) {
    const int lane = threadIdx.x & 31;
    const bool b4 = lane & 16, b3 = lane & 8;
    const float r0 = __fadd_rn(b4 ? v[2] : v[0], __shfl_xor_sync(0xffffffffu, b4 ? v[0] : v[2], 16));
    const float r1 = __fadd_rn(b4 ? 0.0f : v[1], __shfl_xor_sync(0xffffffffu, b4 ? v[1] : 0.0f, 16));
    float r = __fadd_rn(b3 ? r1 : r0, __shfl_xor_sync(0xffffffffu, b3 ? r0 : r1, 8));
#pragma unroll
    for (int m = 4; m >= 1; m >>= 1) r = __fadd_rn(r, __shfl_xor_sync(0xffffffffu, r, m));
    return r;
}

constexpr int kSlots = 2;  // two rows in flight a CTA (about four CTAs a SM)

// PV elements a load, NV loads a thread; FULL: the threads' groups are exactly the
// row's.  slots > 0: rows come through a ring of that many slots of x and dy.
// partial: [gridDim.x][cols] of dgamma followed by the same of dbeta (null: not
// wanted).  dx may be null.
template <typename T, typename GT, int PV, int NV, bool RING, bool FULL>
__global__ void __launch_bounds__(PV * NV > 16 ? 256 : 512)
    k_layer_norm_bwd(const T* __restrict__ x, const GT* __restrict__ gamma, const T* __restrict__ dy,
                     T* __restrict__ dx, float* __restrict__ partial, int64_t rows, int cols, float eps, int slots,
                     int* status) {
    pdl_begin();
    using C = Cols<T, PV, NV>;
    using V = typename C::V;
    extern __shared__ __align__(16) unsigned char ring[];  // slots x (a row of x, a row of dy), then gamma (WIDE)
    __shared__ uint64_t bars[kSlots];
    __shared__ float sum1[32], sum3[3][32];  // by warp; those past the last one stay 0
    const int t = threadIdx.x, th = blockDim.x, lane = t & 31, w = t >> 5;
    const int packs = cols / PV;
    int span = 1;  // the warps, up to a power of two
    while (span < th >> 5) span *= 2;
    if (t < 32) {
        sum1[t] = 0.0f;
        sum3[0][t] = sum3[1][t] = sum3[2][t] = 0.0f;
    }
    const int64_t G = gridDim.x;
    const uint32_t row_bytes = static_cast<uint32_t>(cols * sizeof(T));
    const uint32_t bar0 = rowpipe::smem_addr(bars), ring0 = rowpipe::smem_addr(ring);
    auto fill = [&](int slot, int64_t row) {
        const uint32_t bar = bar0 + 8u * slot, at = ring0 + slot * 2 * row_bytes;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(2 * row_bytes) : "memory");
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(at),
                     "l"(x + row * cols), "r"(row_bytes), "r"(bar)
                     : "memory");
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                         at + row_bytes),
                     "l"(dy + row * cols), "r"(row_bytes), "r"(bar)
                     : "memory");
    };
    long long limit = 0;
    if constexpr (RING) {
        limit = wait_limit(status);
        if (t == 0) {
            for (int s = 0; s < slots; ++s)
                asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar0 + 8u * s) : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            for (int s = 0; s < slots; ++s)
                if (blockIdx.x + s * G < rows) fill(s, blockIdx.x + s * G);
        }
    }
    RowWork<T, PV, NV, FULL> work;
    work.begin(gamma, reinterpret_cast<float4*>(ring + 2 * slots * row_bytes), t, th, packs);
    const float inv_n = __frcp_rn(static_cast<float>(cols));
    __syncthreads();
    C nx, ny;  // !RING: the next row; columns past the end stay 0
    auto load = [&](const V* xr, const V* yr, C& a, C& b) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (work.in(i)) {
                a.v[i] = xr[t + i * th];
                b.v[i] = yr[t + i * th];
            }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < PV; ++e) {
            from_f(0.0f, nx.v[i].v[e]);
            from_f(0.0f, ny.v[i].v[e]);
        }
    auto row_at = [&](const T* p, int64_t r) { return reinterpret_cast<const V*>(p + r * cols); };
    if (!RING) load(row_at(x, blockIdx.x), row_at(dy, blockIdx.x), nx, ny);
    int slot = 0;
    uint32_t parity = 0;
    bool ok = true;
    for (int64_t row = blockIdx.x; row < rows; row += G) {
        bool landed = true;
        if constexpr (RING) {
            landed = rowpipe::bar_wait(bar0 + 8u * slot, parity, limit);
            const V* at = reinterpret_cast<const V*>(ring + slot * 2 * row_bytes);
            if (landed) load(at, at + packs, nx, ny);
        }
        const float s = warp_add(work.take(nx, ny));
        if (!RING && row + G < rows) load(row_at(x, row + G), row_at(dy, row + G), nx, ny);
        if (lane == 0) sum1[w] = s;
        // every thread has its part of the row, and of the row before it all sums
        if constexpr (RING) {
            if (__syncthreads_or(!landed)) {
                ok = false;
                break;
            }
            const int64_t next = row + slots * G;
            if (t == 0 && next < rows) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                fill(slot, next);
            }
        } else {
            __syncthreads();
        }
        float mean = sum1[lane & (span - 1)];
        for (int m = span / 2; m >= 1; m >>= 1) mean = __fadd_rn(mean, __shfl_xor_sync(0xffffffffu, mean, m));
        mean = __fmul_rn(mean, inv_n);
        float s3[3];
        work.deviations(mean, s3);
        const float mine = warp_sum3(s3);
        if ((lane & 7) == 0 && lane < 24) sum3[lane >> 3][w] = mine;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            s3[k] = sum3[k][lane & (span - 1)];
            for (int m = span / 2; m >= 1; m >>= 1) s3[k] = __fadd_rn(s3[k], __shfl_xor_sync(0xffffffffu, s3[k], m));
        }
        C out;
        work.outputs(s3, inv_n, eps, out);
        if (dx) {
            V* dr = reinterpret_cast<V*>(dx + row * cols);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (work.in(i)) dr[t + i * th] = out.v[i];
        }
        if (RING && ++slot == slots) {
            slot = 0;
            parity ^= 1u;
        }
    }
    if (RING && !ok) {
        // the copies still in flight -- of this slot's row and those after it -- land first
        if (t == 0) {
            atomicExch(status, QSML_E_TIMEOUT);
            for (int k = 0; k < slots; ++k) {
                rowpipe::bar_drain(bar0 + 8u * slot, parity);
                if (++slot == slots) {
                    slot = 0;
                    parity ^= 1u;
                }
            }
        }
        __syncthreads();
    }
    if (!partial) return;
    float* pg = partial + blockIdx.x * static_cast<int64_t>(cols);
    float* pb = pg + G * cols;
    if constexpr (PV >= 4) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (work.in(i))
#pragma unroll
                for (int q = 0; q < PV / 4; ++q) {
                    const int j = (i * PV + q * 4) / 2, c = (t + i * th) * PV + q * 4;
                    const float2 a0 = unpack(work.sg[j]), a1 = unpack(work.sg[j + 1]);
                    const float2 b0 = unpack(work.sb[j]), b1 = unpack(work.sb[j + 1]);
                    *reinterpret_cast<float4*>(pg + c) = make_float4(a0.x, a0.y, a1.x, a1.y);
                    *reinterpret_cast<float4*>(pb + c) = make_float4(b0.x, b0.y, b1.x, b1.y);
                }
    } else {
#pragma unroll
        for (int j = 0; j < C::H; ++j) {
            const float2 a = unpack(work.sg[j]), b = unpack(work.sb[j]);
            const int i0 = 2 * j / PV, i1 = (2 * j + 1) / PV;
            const int c0 = (t + i0 * th) * PV + 2 * j % PV, c1 = (t + i1 * th) * PV + (2 * j + 1) % PV;
            if (work.in(i0)) {
                pg[c0] = a.x;
                pb[c0] = b.x;
            }
            if (work.in(i1)) {
                pg[c1] = a.y;
                pb[c1] = b.y;
            }
        }
    }
}

// Narrow rows: L lanes a row, so 32 / L rows a warp and 8 warps a CTA, no barrier
// between them; the next row's loads are in flight while this one is reduced.
template <typename T, typename GT, int PV, int NV, int L>
__global__ void __launch_bounds__(256)
    k_layer_norm_bwd_groups(const T* __restrict__ x, const GT* __restrict__ gamma, const T* __restrict__ dy,
                            T* __restrict__ dx, float* __restrict__ partial, int64_t rows, int cols, float eps) {
    pdl_begin();
    using C = Cols<T, PV, NV>;
    using V = typename C::V;
    extern __shared__ float fold[];  // the warps' column sums, [2][cols]
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, t = lane % L;
    const int packs = cols / PV;
    RowWork<T, PV, NV, false> work;
    work.begin(gamma, nullptr, t, L, packs);
    const float inv_n = __frcp_rn(static_cast<float>(cols));
    C nx, ny;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < PV; ++e) {
            from_f(0.0f, nx.v[i].v[e]);
            from_f(0.0f, ny.v[i].v[e]);
        }
    auto load = [&](int64_t r) {
        const V* xr = reinterpret_cast<const V*>(x + r * cols);
        const V* yr = reinterpret_cast<const V*>(dy + r * cols);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (work.in(i)) {
                nx.v[i] = xr[t + i * L];
                ny.v[i] = yr[t + i * L];
            }
    };
    auto group_sum = [](float v) {
#pragma unroll
        for (int m = L / 2; m >= 1; m >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, m));
        return v;
    };
    constexpr int PER = 32 / L;  // rows a warp
    const int64_t step = static_cast<int64_t>(gridDim.x) * 8 * PER;
    // the warp's first row decides the trips, so that all lanes take part in the sums
    int64_t first = (static_cast<int64_t>(blockIdx.x) * 8 + w) * PER;
    if (first + lane / L < rows) load(first + lane / L);
    for (; first < rows; first += step) {
        const int64_t row = first + lane / L;
        const bool here = row < rows;
        float s3[3];
        const float s = work.take(nx, ny);
        if (row + step < rows) load(row + step);
        work.deviations(__fmul_rn(group_sum(s), inv_n), s3);
#pragma unroll
        for (int k = 0; k < 3; ++k) s3[k] = group_sum(s3[k]);
        if (here) {  // a group past the last row adds nothing to the columns' sums
            C out;
            work.outputs(s3, inv_n, eps, out);
            if (dx) {
                V* dr = reinterpret_cast<V*>(dx + row * cols);
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (work.in(i)) dr[t + i * L] = out.v[i];
            }
        }
    }
    if (!partial) return;
    // the groups of a warp by exchanges, then the warps one after another
#pragma unroll
    for (int m = L; m < 32; m <<= 1)
#pragma unroll
        for (int j = 0; j < C::H; ++j) {
            P2 a, b;
            a.v = __shfl_xor_sync(0xffffffffu, work.sg[j].v, m);
            b.v = __shfl_xor_sync(0xffffffffu, work.sb[j].v, m);
            work.sg[j] = add2(work.sg[j], a);
            work.sb[j] = add2(work.sb[j], b);
        }
    for (int k = 0; k < 8; ++k) {
        if (w == k && lane < L) {
#pragma unroll
            for (int j = 0; j < C::H; ++j) {
                const float2 a = unpack(work.sg[j]), b = unpack(work.sb[j]);
                const float va[2] = {a.x, a.y}, vb[2] = {b.x, b.y};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int i = (2 * j + h) / PV, c = (t + i * L) * PV + (2 * j + h) % PV;
                    if (work.in(i)) {
                        fold[c] = k ? __fadd_rn(fold[c], va[h]) : va[h];
                        fold[cols + c] = k ? __fadd_rn(fold[cols + c], vb[h]) : vb[h];
                    }
                }
            }
        }
        __syncthreads();
    }
    float* pg = partial + blockIdx.x * static_cast<int64_t>(cols);
    float* pb = pg + gridDim.x * static_cast<int64_t>(cols);
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
        pg[c] = fold[c];
        pb[c] = fold[cols + c];
    }
}

// PV values of gamma, which lies at a 16-byte boundary for PV > 1 (single loads of
// neighbouring lanes lie PV apart: 4096 x 16384 of binary16 took 244 us, now 154).
template <typename GT, int PV> __device__ __forceinline__ void gammas(const GT* g, float (&o)[PV]) {
    constexpr int W = 16 / sizeof(GT) < PV ? 16 / sizeof(GT) : PV;
#pragma unroll
    for (int i = 0; i < PV / W; ++i) {
        const Vec<GT, W> v = reinterpret_cast<const Vec<GT, W>*>(g)[i];
#pragma unroll
        for (int e = 0; e < W; ++e) o[i * W + e] = to_f(v.v[e]);
    }
}

// Rows of any width, a CTA a row; leaves the row's mean and rstd for the column kernel.
// NV > 0: the threads hold the row, NV loads of PV elements each; NV == 0: three sweeps
// over global memory (L2 holds a row between them).
template <typename T, typename GT, int PV, int NV>
__global__ void __launch_bounds__(512)
    k_layer_norm_bwd_rows(const T* __restrict__ x, const GT* __restrict__ gamma, const T* __restrict__ dy,
                          T* __restrict__ dx, float2* __restrict__ stats, int64_t rows, int cols, float eps) {
    pdl_begin();
    using V = Vec<T, PV>;
    constexpr int HELD = NV > 0 ? NV : 1;
    __shared__ float slots[4 * 32];
    const float inv_n = __frcp_rn(static_cast<float>(cols));
    const unsigned packs = cols / PV;  // a step past 2^31 - 1 columns still fits
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const V* xr = reinterpret_cast<const V*>(x + row * cols);
        const V* yr = reinterpret_cast<const V*>(dy + row * cols);
        V* dr = dx ? reinterpret_cast<V*>(dx + row * cols) : nullptr;
        V xh[HELD], yh[HELD];
        // f(p, x, dy) for this thread's loads p
        auto sweep = [&](auto&& f) {
            if constexpr (NV > 0) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (threadIdx.x + i * 512 < packs) f(threadIdx.x + i * 512, xh[i], yh[i]);
            } else {
#pragma unroll 2
                for (unsigned p = threadIdx.x; p < packs; p += 512) {
                    const V v = xr[p], y = yr[p];
                    f(p, v, y);
                }
            }
        };
        float s1[1] = {0.0f};
        auto add = [&](const V& v) {
#pragma unroll
            for (int e = 0; e < PV; ++e) s1[0] = __fadd_rn(s1[0], to_f(v.v[e]));
        };
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (threadIdx.x + i * 512 < packs) {
                    xh[i] = xr[threadIdx.x + i * 512];
                    yh[i] = yr[threadIdx.x + i * 512];
                }
            sweep([&](unsigned, const V& v, const V&) { add(v); });
        } else {
#pragma unroll 4
            for (unsigned p = threadIdx.x; p < packs; p += 512) add(xr[p]);
        }
        row_sums(s1, slots);
        const float mean = __fmul_rn(s1[0], inv_n);
        float s3[3] = {0.0f, 0.0f, 0.0f};
        sweep([&](unsigned p, const V& v, const V& y) {
            float g[PV];
            gammas<GT, PV>(gamma + p * PV, g);
#pragma unroll
            for (int e = 0; e < PV; ++e) {
                const float d = __fsub_rn(to_f(v.v[e]), mean), h = __fmul_rn(to_f(y.v[e]), g[e]);
                s3[0] = __fmaf_rn(d, d, s3[0]);
                s3[1] = __fadd_rn(s3[1], h);
                s3[2] = __fmaf_rn(h, d, s3[2]);
            }
        });
        row_sums(s3, slots + 32);
        const float rstd = rsqrtf(__fmaf_rn(s3[0], inv_n, eps));
        if (stats && threadIdx.x == 0) stats[row] = make_float2(mean, rstd);
        if (!dx) continue;
        const float a = __fmul_rn(__fmul_rn(s3[1], inv_n), rstd);
        const float b = __fmul_rn(__fmul_rn(__fmul_rn(s3[2], inv_n), rstd), __fmul_rn(rstd, rstd));
        sweep([&](unsigned p, const V& v, const V& y) {
            float g[PV];
            gammas<GT, PV>(gamma + p * PV, g);
            V o;
#pragma unroll
            for (int e = 0; e < PV; ++e) {
                const float d = __fsub_rn(to_f(v.v[e]), mean), h = __fmul_rn(to_f(y.v[e]), g[e]);
                from_f(__fmaf_rn(h, rstd, -__fmaf_rn(d, b, a)), o.v[e]);
            }
            dr[p] = o;
        });
    }
}

// Column sums of dy xh and dy over the rows [blockIdx.y * chunk, + chunk): a
// thread PV columns.
template <typename T, int PV>
__global__ void __launch_bounds__(128)
    k_layer_norm_bwd_cols(const T* __restrict__ x, const T* __restrict__ dy, const float2* __restrict__ stats,
                          float* __restrict__ partial, int64_t rows, int cols, int64_t chunk) {
    pdl_begin();
    using V = Vec<T, PV>;
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x) * PV;
    if (c >= cols) return;
    const int64_t r0 = blockIdx.y * chunk, r1 = r0 + chunk < rows ? r0 + chunk : rows;
    float sg[PV], sb[PV];
#pragma unroll
    for (int e = 0; e < PV; ++e) sg[e] = sb[e] = 0.0f;
#pragma unroll 4
    for (int64_t r = r0; r < r1; ++r) {
        const float2 st = stats[r];
        const V v = *reinterpret_cast<const V*>(x + r * cols + c), y = *reinterpret_cast<const V*>(dy + r * cols + c);
#pragma unroll
        for (int e = 0; e < PV; ++e) {
            const float f = to_f(y.v[e]);
            sg[e] = __fmaf_rn(f, __fmul_rn(__fsub_rn(to_f(v.v[e]), st.x), st.y), sg[e]);
            sb[e] = __fadd_rn(sb[e], f);
        }
    }
    float* pg = partial + blockIdx.y * static_cast<int64_t>(cols) + c;
    float* pb = pg + gridDim.y * static_cast<int64_t>(cols);
#pragma unroll
    for (int e = 0; e < PV; ++e) {
        pg[e] = sg[e];
        pb[e] = sb[e];
    }
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

// CTAs of `kernel` a SM, once per device, block size and shared memory; opts in to
// that much dynamic shared memory.
qsml_status_t resident(Context* ctx, const void* kernel, int block, size_t smem, int* per_sm) {
    static std::mutex mu;
    static std::map<std::pair<std::pair<const void*, int>, std::pair<int, size_t>>, int> known;
    static std::map<std::pair<const void*, int>, size_t> opted;
    std::lock_guard<std::mutex> lk(mu);
    size_t& have = opted[{kernel, ctx->device}];
    if (smem > 40 * 1024 && smem > have) {  // 48 KiB without it, static memory included
        QSML_TRY_STATUS(check_cuda(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                             static_cast<int>(smem)),
                                   "layer norm backward: shared-memory attribute"));
        have = smem;
    }
    int& n = known[{{kernel, ctx->device}, {block, smem}}];
    if (n == 0) {
        QSML_TRY_STATUS(check_cuda(ctx, cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, block, smem),
                                   "layer norm backward: occupancy"));
        if (n < 1) n = 1;
    }
    *per_sm = n;
    return QSML_OK;
}

template <typename T, typename GT, int PV, int NV, bool RING, bool FULL>
qsml_status_t launch_cta(Context* ctx, const Args& a, int th) {
    auto kernel = k_layer_norm_bwd<T, GT, PV, NV, RING, FULL>;
    const size_t slot = 2 * static_cast<size_t>(a.cols) * sizeof(T);
    const int slots = RING ? kSlots : 0;
    const size_t smem = slots * slot + (PV * NV > 16 ? a.cols * sizeof(float) : 0);
    int per_sm = 0;
    QSML_TRY_STATUS(resident(ctx, reinterpret_cast<const void*>(kernel), th, smem, &per_sm));
    int64_t grid = static_cast<int64_t>(ctx->num_sms) * per_sm;
    if (grid > a.rows) grid = a.rows;
    Workspace ws(ctx);
    void* partial = nullptr;
    if (a.sums()) QSML_TRY_STATUS(ws.get(static_cast<size_t>(grid) * a.cols * 2 * sizeof(float), &partial));
    const cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(grid)), dim3(th), smem, ctx->stream,
                                     static_cast<const T*>(a.x), static_cast<const GT*>(a.gamma),
                                     static_cast<const T*>(a.dy), static_cast<T*>(a.dx), static_cast<float*>(partial),
                                     a.rows, static_cast<int>(a.cols), a.eps, slots, ctx->status);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_layer_norm_bwd");
    QSML_TRY_STATUS(after_launch(ctx, "k_layer_norm_bwd"));
    return a.sums() ? finish(ctx, a, static_cast<float*>(partial), grid) : QSML_OK;
}

template <typename T, typename GT, int PV, int NV, int L> qsml_status_t launch_groups(Context* ctx, const Args& a) {
    auto kernel = k_layer_norm_bwd_groups<T, GT, PV, NV, L>;
    const size_t smem = a.sums() ? static_cast<size_t>(a.cols) * 2 * sizeof(float) : 0;
    int per_sm = 0;
    QSML_TRY_STATUS(resident(ctx, reinterpret_cast<const void*>(kernel), 256, smem, &per_sm));
    int64_t grid = static_cast<int64_t>(ctx->num_sms) * per_sm;
    const int64_t most = (a.rows + 8 * (32 / L) - 1) / (8 * (32 / L));
    if (grid > most) grid = most;
    Workspace ws(ctx);
    void* partial = nullptr;
    if (a.sums()) QSML_TRY_STATUS(ws.get(static_cast<size_t>(grid) * a.cols * 2 * sizeof(float), &partial));
    const cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(grid)), dim3(256), smem, ctx->stream,
                                     static_cast<const T*>(a.x), static_cast<const GT*>(a.gamma),
                                     static_cast<const T*>(a.dy), static_cast<T*>(a.dx), static_cast<float*>(partial),
                                     a.rows, static_cast<int>(a.cols), a.eps);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_layer_norm_bwd_groups");
    QSML_TRY_STATUS(after_launch(ctx, "k_layer_norm_bwd_groups"));
    return a.sums() ? finish(ctx, a, static_cast<float*>(partial), grid) : QSML_OK;
}

template <typename T, typename GT, int PV>
qsml_status_t launch_wide_bwd(Context* ctx, const Args& a) {
    Workspace ws(ctx);
    void *stats = nullptr, *partial = nullptr;
    // a chunk of rows for each CTA of the column kernel, about eight CTAs an SM, at least 16
    // rows (with fewer the partial sums cost more than the rows)
    const int64_t tiles = (a.cols / PV + 127) / 128;
    int64_t parts = (8 * ctx->num_sms + tiles - 1) / tiles;
    const int64_t most = (a.rows + 15) / 16;
    if (parts > most) parts = most;
    const int64_t chunk = (a.rows + parts - 1) / parts;
    parts = (a.rows + chunk - 1) / chunk;
    if (a.sums()) {
        QSML_TRY_STATUS(ws.get(static_cast<size_t>(a.rows) * sizeof(float2), &stats));
        QSML_TRY_STATUS(ws.get(static_cast<size_t>(parts) * a.cols * 2 * sizeof(float), &partial));
    }
    const int64_t grid = a.rows < 4 * ctx->num_sms ? a.rows : 4 * ctx->num_sms;
    // the row in registers where 512 threads hold it, unless that costs resident CTAs that
    // many binary32 rows need (148 x 16384: 35 us in sweeps, 28 held; 4096 x 10000: 161 and
    // 190; binary16 4096 x 10000: 177 and 113)
    const int64_t packs = a.cols / PV;
    constexpr int FEW = PV == 8 ? 4 : 0, MANY = PV == 1 ? 16 : 8;
    auto kernel = k_layer_norm_bwd_rows<T, GT, PV, 0>;
    if (sizeof(T) == 2 || a.rows <= 4 * ctx->num_sms) {
        if (packs <= FEW * 512) kernel = k_layer_norm_bwd_rows<T, GT, PV, FEW>;
        else if (packs <= MANY * 512) kernel = k_layer_norm_bwd_rows<T, GT, PV, MANY>;
    }
    cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(grid)), dim3(512), 0, ctx->stream,
                               static_cast<const T*>(a.x), static_cast<const GT*>(a.gamma),
                               static_cast<const T*>(a.dy), static_cast<T*>(a.dx), static_cast<float2*>(stats), a.rows,
                               static_cast<int>(a.cols), a.eps);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_layer_norm_bwd_rows");
    QSML_TRY_STATUS(after_launch(ctx, "k_layer_norm_bwd_rows"));
    if (!a.sums()) return QSML_OK;
    e = launch_pdl(k_layer_norm_bwd_cols<T, PV>, dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(parts)),
                   dim3(128), 0, ctx->stream, static_cast<const T*>(a.x), static_cast<const T*>(a.dy),
                   static_cast<const float2*>(stats), static_cast<float*>(partial), a.rows, static_cast<int>(a.cols), chunk);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_layer_norm_bwd_cols");
    QSML_TRY_STATUS(after_launch(ctx, "k_layer_norm_bwd_cols"));
    return finish(ctx, a, static_cast<float*>(partial), parts);
}

// The threads of a CTA that hold a row's groups, NV each, and whether exactly.
template <typename T, typename GT, int PV, int NV, bool RING> qsml_status_t run_cta(Context* ctx, const Args& a) {
    const int64_t packs = a.cols / PV;
    const int th = static_cast<int>(((packs + NV - 1) / NV + 31) / 32 * 32);
    if (RING && packs == th * NV) return launch_cta<T, GT, PV, NV, RING, RING>(ctx, a, th);
    return launch_cta<T, GT, PV, NV, RING, false>(ctx, a, th);
}

// Loads of PV elements.  Rows of up to 512 columns: 4 to 32 lanes with 16 elements
// each.  Up to 8192: a CTA, whose threads hold 32 elements of binary16 rows (fewer
// warps meet at the row's two barriers and more rows are on a SM: 16384 x 4096 took
// 93 us so, 98 with 16 elements, 124 with 8), 16 of binary32 ones.  Single elements:
// 8 a thread, 12 up to 6144 columns (with 16 the compiler runs out of the registers of
// 512 threads: 6007 x 6001 binary32 took 387 us, with 12 90), then the two kernels
// (6007 x 8191 binary32: 283 us; with 16 a thread 415).
template <typename T, typename GT, int PV> qsml_status_t pick(Context* ctx, const Args& a) {
    const int64_t packs = a.cols / PV;
    if (a.cols <= 512) {
        constexpr int NV = 16 / PV;
        if (packs <= 4 * NV) return launch_groups<T, GT, PV, NV, 4>(ctx, a);
        if (packs <= 8 * NV) return launch_groups<T, GT, PV, NV, 8>(ctx, a);
        if (packs <= 16 * NV) return launch_groups<T, GT, PV, NV, 16>(ctx, a);
        return launch_groups<T, GT, PV, NV, 32>(ctx, a);
    }
    if (a.cols > (PV == 1 ? 6144 : 8192)) return launch_wide_bwd<T, GT, PV>(ctx, a);
    if constexpr (PV == 1)
        return a.cols <= 4096 ? run_cta<T, GT, 1, 8, false>(ctx, a) : run_cta<T, GT, 1, 12, false>(ctx, a);
    else
        return run_cta<T, GT, PV, (sizeof(T) == 2 ? 32 : 16) / PV, true>(ctx, a);
}

template <typename T, typename GT>
qsml_status_t run_bwd(Context* ctx, const Args& a) {
    constexpr int PV = 16 / sizeof(T);
    if (a.cols % PV == 0 && aligned16(a.x) && aligned16(a.dy) && (!a.dx || aligned16(a.dx)) &&
        (a.cols <= 8192 || aligned16(a.gamma)))
        return pick<T, GT, PV>(ctx, a);
    return pick<T, GT, 1>(ctx, a);
}

}  // namespace
}  // namespace qsml

using namespace qsml;

extern "C" qsml_status_t qsml_layer_norm_backward(qsml_ctx* handle, const qsml_tdesc* x, const qsml_tdesc* gamma,
                                                  const qsml_tdesc* dy, float eps, const qsml_tdesc* dx,
                                                  const qsml_tdesc* dgamma, const qsml_tdesc* dbeta) try {
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
} QSML_NO_THROW
