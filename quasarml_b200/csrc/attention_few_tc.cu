// Attention of few queries over many keys in binary16, heads of up to 128 columns: the next
// tokens of sequences over their caches, 16 rows (heads of a group and queries) a CTA.
//
// Bound by HBM.  16 rows would leave seven eighths of a tcgen05 tile empty and their scores would
// go through TMEM; mma.sync's 16 x 8 tiles hold them in the registers that compute the exponentials,
// at a rate that is several times what the cache's bytes need.  Each warp goes over tiles of KT keys
// of its own through a ring that only it fills (cp.async, 16 bytes a lane, the units of a row
// permuted by the row so that ldmatrix meets no bank twice), so there is no barrier until the
// warps' sums are joined at the end; parts of a row's keys are joined as in attention_few.cu.
// P is 2^(s c - m c + 8), which keeps small weights in binary16's normal range.  Measured: 64 sequences
// over 2048 keys of 16 heads of 64 (537 MB) 90 us, 0.91 of the copy's rate; 16 over 1 to 8192 keys of 8 heads
// of 128 (304 MB) 73 us, with their first loads and last joins in the open.
#include <algorithm>

#include "attention.cuh"

namespace qsml {
namespace attn {
namespace {

constexpr int kThreads = 128, kWarps = 4, KT = 16, STAGES = 2;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, SHIFT = 8.0f;

template <int DP> struct Shape {
    static constexpr int ROW = DP * 2, TILE = KT * ROW;  // bytes
    static constexpr int STAGE = 2 * TILE;               // K and V
    static constexpr size_t RING = size_t(kWarps) * STAGES * STAGE, JOIN = sizeof(float) * kWarps * (16 * DP + 32);
    static constexpr size_t SMEM = RING > JOIN ? RING : JOIN;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

// The visible keys [n0, n0 + KT) below end of K and V into a stage; zeros elsewhere.  By one warp.
template <int DP>
__device__ __forceinline__ void load_stage(uint32_t dst, const Problem& p, const __half* k, const __half* v, const Keys& keys, int n0, int end) {
    constexpr int UNITS = DP / 8, ROWS = 32 / UNITS;  // 16-byte units a row, rows at once
    const int lane = threadIdx.x & 31, unit = lane % UNITS;
#pragma unroll
    for (int i = 0; i < KT / ROWS; ++i) {
        const int r = lane / UNITS + i * ROWS, n = n0 + r;
        const bool in = n < end && unit * 8 < p.D;
        const int64_t key = in ? keys.key(n) : 0;
        const uint32_t to = dst + r * Shape<DP>::ROW + ((unit ^ (r & 7)) << 4);
        const int bytes = in ? 16 : 0;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(in ? k + key * p.k.s + unit * 8 : k), "r"(bytes) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + Shape<DP>::TILE), "l"(in ? v + key * p.v.s + unit * 8 : v), "r"(bytes) : "memory");
    }
}

template <int DP>
__global__ void __launch_bounds__(kThreads) k_attention_few_tc(const __grid_constant__ Problem p, Parts parts, int row_tiles) {
    using S = Shape<DP>;
    extern __shared__ __align__(128) unsigned char smem[];
    pdl_begin();
    const int part = blockIdx.x % parts.parts, group = blockIdx.x / parts.parts;
    const int rt = group % row_tiles, hk = group / row_tiles % p.Hk, b = group / row_tiles / p.Hk;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, col = lane & 3;
    const Seq seq(p, b);
    const int off = seq.nk - seq.nq, R = p.Sq * p.G, r0 = rt * 16;
    const int first = r0 / p.G, last = min((min(r0 + 16, R) - 1) / p.G, seq.nq - 1);  // queries of the rows
    const Keys keys(p, seq.nk, first + off, last + off);
    const int all = first < seq.nq ? keys.count() : 0;
    const int share = (all + parts.parts - 1) / parts.parts;
    const int n0 = min(part * share, all), n1 = min(n0 + share, all);
    const __half* k = reinterpret_cast<const __half*>(p.k.p) + b * p.k.b + hk * p.k.h;
    const __half* v = reinterpret_cast<const __half*>(p.v.p) + b * p.v.b + hk * p.v.h;
    const uint32_t ring = smem_u32(smem) + warp * STAGES * S::STAGE;
    // this warp's tiles: every fourth of the part
    const int tiles = n1 > n0 + warp * KT ? (n1 - n0 - warp * KT + kWarps * KT - 1) / (kWarps * KT) : 0;
    auto begin = [&](int i) {
        if (i < tiles) load_stage<DP>(ring + i % STAGES * S::STAGE, p, k, v, keys, n0 + (i * kWarps + warp) * KT, n1);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int i = 0; i < STAGES - 1; ++i) begin(i);

    // rows quad and quad + 8 of the 16: their queries (nq: none) and Q as the A operand
    int query[2];
    uint32_t a[DP / 16][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = r0 + quad + 8 * i;
        const bool in = r < R && r / p.G < seq.nq;
        query[i] = in ? r / p.G : seq.nq;
        const __half* q = reinterpret_cast<const __half*>(p.q.p) + (in ? b * p.q.b + r / p.G * p.q.s + (hk * p.G + r % p.G) * p.q.h : 0);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = s * 16 + h * 8 + col * 2;
                a[s][i + 2 * h] = in && c < p.D ? *reinterpret_cast<const uint32_t*>(q + c) : 0u;
            }
    }
    const float c = p.scale * kLog2e;
    const int first_pos = first + off, last_pos = last + off;
    float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (auto& x : o) x[0] = x[1] = x[2] = x[3] = 0.0f;
    for (int i = 0; i < tiles; ++i) {
        begin(i + STAGES - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
        const uint32_t kt = ring + i % STAGES * S::STAGE, vt = kt + S::TILE;
        float s[KT / 8][4];
#pragma unroll
        for (auto& x : s) x[0] = x[1] = x[2] = x[3] = 0.0f;
        // a lane's row of the matrices: keys 8 (lane / 16) + lane % 8, columns 8 (lane / 8 % 2) on
        const int kr = (lane >> 4) * 8 + (lane & 7);
#pragma unroll
        for (int t = 0; t < KT / 16; ++t)
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                uint32_t r[4];
                ldmatrix4(r, kt + (t * 16 + kr) * S::ROW + (((2 * d + (lane >> 3 & 1)) ^ (kr & 7)) << 4));
                mma(s[2 * t], a[d], r[0], r[1]);
                mma(s[2 * t + 1], a[d], r[2], r[3]);
            }
        const int n = n0 + (i * kWarps + warp) * KT;
        // whether every row sees every key of the tile
        const int low = keys.key(n), high = keys.key(n + KT - 1);
        const bool whole = n + KT <= n1 && high <= first_pos && (p.window == 0 || last_pos - low < p.window || high < p.sinks) &&
                           query[0] < seq.nq && query[1] < seq.nq;
        if (!__all_sync(0xffffffffu, whole)) {
#pragma unroll
            for (int t = 0; t < KT / 8; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = n + t * 8 + col * 2 + (e & 1), qi = query[e >> 1];
                    if (!(at < n1 && qi < seq.nq && sees(p, qi + off, keys.key(at)))) s[t][e] = -INFINITY;
                }
        }
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < KT / 8; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], s[t][e]);
        float f[2], ref[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float now = fmaxf(m[h], quad_max(top[h]) * c);
            const float base = now == -INFINITY ? 0.0f : now;
            f[h] = exp2f(m[h] - base);
            ref[h] = SHIFT - base;
            m[h] = now;
            l[h] *= f[h];
        }
        if (__any_sync(0xffffffffu, f[0] != 1.0f || f[1] != 1.0f)) {
#pragma unroll
            for (auto& x : o) x[0] *= f[0], x[1] *= f[0], x[2] *= f[1], x[3] *= f[1];
        }
        uint32_t w[KT / 8][2];
#pragma unroll
        for (int t = 0; t < KT / 8; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float x = exp2f(fmaf(s[t][2 * h], c, ref[h])), y = exp2f(fmaf(s[t][2 * h + 1], c, ref[h]));
                l[h] += x + y;
                const __half2 z = __floats2half2_rn(x, y);
                w[t][h] = *reinterpret_cast<const uint32_t*>(&z);
            }
        const int vr = lane & 15;
#pragma unroll
        for (int t = 0; t < KT / 16; ++t) {
            const uint32_t pa[4] = {w[2 * t][0], w[2 * t][1], w[2 * t + 1][0], w[2 * t + 1][1]};
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                uint32_t r[4];
                ldmatrix4_t(r, vt + (t * 16 + vr) * S::ROW + (((2 * d + (lane >> 4)) ^ (vr & 7)) << 4));
                mma(o[2 * d], pa, r[0], r[1]);
                mma(o[2 * d + 1], pa, r[2], r[3]);
            }
        }
        __syncwarp();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // the warps' sums, in their order
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    __syncthreads();
    float *so = reinterpret_cast<float*>(smem), *st = so + kWarps * 16 * DP;  // [warps][16][DP], [warps][16][2]
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = warp * 16 + quad + 8 * h;
#pragma unroll
        for (int t = 0; t < DP / 8; ++t) *reinterpret_cast<float2*>(so + r * DP + t * 8 + col * 2) = make_float2(o[t][2 * h], o[t][2 * h + 1]);
        if (col == 0) st[2 * r] = m[h], st[2 * r + 1] = l[h];
    }
    __syncthreads();
    const float unshift = exp2f(-SHIFT);
    for (int r = warp; r < 16 && r0 + r < R; r += kWarps) {
        const int q = (r0 + r) / p.G, h = hk * p.G + (r0 + r) % p.G;
        const int64_t row = (static_cast<int64_t>(b) * p.Hq + h) * p.Sq + q;
        float top = -INFINITY, norm = 0.0f, g[kWarps];
#pragma unroll
        for (int i = 0; i < kWarps; ++i) top = fmaxf(top, st[2 * (i * 16 + r)]);
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            g[i] = exp2f(st[2 * (i * 16 + r)] - (top == -INFINITY ? 0.0f : top)) * unshift;
            norm = fmaf(st[2 * (i * 16 + r) + 1], g[i], norm);
        }
        const bool any = norm > 0.0f || isnan(norm);
        const float f = parts.parts > 1 ? 1.0f : any ? 1.0f / norm : 0.0f;
        for (int d = lane * 2; d < p.D; d += 64) {
            float2 x = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                const float2 y = *reinterpret_cast<const float2*>(so + (i * 16 + r) * DP + d);
                x.x = fmaf(y.x, g[i], x.x);
                x.y = fmaf(y.y, g[i], x.y);
            }
            if (parts.parts > 1)
                *reinterpret_cast<float2*>(parts.sum + (row * parts.parts + part) * p.D + d) = x;
            else
                *reinterpret_cast<__half2*>(reinterpret_cast<__half*>(p.o.p) + b * p.o.b + q * p.o.s + h * p.o.h + d) = __floats2half2_rn(x.x * f, x.y * f);
        }
        if (lane == 0) {
            if (parts.parts > 1) {
                parts.stat[(row * parts.parts + part) * 2] = top;
                parts.stat[(row * parts.parts + part) * 2 + 1] = norm;
            } else if (p.lse) {
                p.lse[row] = any ? (top + log2f(norm)) * kLn2 : -INFINITY;
            }
        }
    }
}

template <int DP> qsml_status_t run(Context* ctx, const Problem& p) {
    const char* name = "k_attention_few_tc";
    const auto kernel = k_attention_few_tc<DP>;
    constexpr size_t smem = Shape<DP>::SMEM;
    QSML_TRY_STATUS(check_cuda(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)), name));
    const int row_tiles = (p.Sq * p.G + 15) / 16;
    const int64_t groups = static_cast<int64_t>(row_tiles) * p.Hk * p.B;
    // A SM holds three CTAs; parts for two are fewer to join: one sequence over 8192 keys 18 us (parts for three
    // 22), over 32768 33 (37), 4 over 4096 23 (24); but 16 over 8192 each 124 (90), whose last wave is short.
    // a warp's accumulators take no more than 8192 keys: they truncate (32768 keys of one sign: 2e-4 of the sum)
    const int64_t n = few_parts(ctx, p, groups, 2, kWarps * KT, kWarps * 8192);
    if (groups * n > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "qsml_attention: dimensions too large");
    Workspace ws(ctx);
    Parts parts;
    QSML_TRY_STATUS(get_parts(ctx, &ws, p, n, &parts));
    const cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(groups * n)), dim3(kThreads), smem, ctx->stream, p, parts, row_tiles);
    if (e != cudaSuccess) return check_cuda(ctx, e, name);
    QSML_TRY_STATUS(after_launch(ctx, name));
    return join_parts(ctx, p, parts);
}

}  // namespace

bool few_tc_takes(const Problem& p) {
    return p.f16 && p.D % 8 == 0 && p.D <= 128 && heads::rows_on(p.k, 2, 16) && heads::rows_on(p.v, 2, 16) && heads::rows_on(p.q, 2, 4) &&
           heads::rows_on(p.o, 2, 4);
}

qsml_status_t forward_few_tc(Context* ctx, const Problem& p) { return p.D <= 64 ? run<64>(ctx, p) : run<128>(ctx, p); }

}  // namespace attn
}  // namespace qsml
