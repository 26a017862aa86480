// Attention of few queries over many keys: the next tokens of sequences over their caches.
//
// Bound by HBM: the visible keys and values are read once, for all heads of a group and all
// queries together (RT rows a CTA).  A sequence's visible keys are split over CTAs so that
// the device is full however few sequences there are; each CTA goes over its part in tiles
// of keys that cp.async brings in while the tile before is used, with the rows' running
// maximum and sum, and leaves its sums and statistics in a workspace that k_attention_join
// adds up in the order of the parts.  With one part there is nothing to join.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention.cuh"
#include "packed.cuh"

namespace qsml {
namespace attn {
namespace {

constexpr int kThreads = 128;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename T, int DP, int RT> struct Shape {
    static constexpr int V = 16 / sizeof(T);
    // keys a tile, in two stages: one CTA a SM for binary32 heads of 256 columns, two to five for the others
    static constexpr int KT = sizeof(T) * DP >= 512 ? 32 : 64;
    static constexpr int LD = DP + V;  // elements between rows: lanes' 16-byte loads 8 by 8 in no bank
    static constexpr int TILE = KT * LD * sizeof(T);
    static constexpr size_t SMEM = 4 * TILE + sizeof(float) * (RT * DP + RT * KT + 3 * RT);
};

// The n-th visible keys [n0, n0 + KT) below end of a head into a tile; zeros elsewhere.
template <typename T, int DP, int RT>
__device__ __forceinline__ void load_keys(unsigned char* dst, const View& v, int64_t at, const Keys& keys, int n0, int end, int D, bool vec) {
    using S = Shape<T, DP, RT>;
    const T* p = reinterpret_cast<const T*>(v.p) + at;
    if (vec) {
        constexpr int C = DP / S::V;
        for (int i = threadIdx.x; i < S::KT * C; i += kThreads) {
            const int r = i / C, c = i % C * S::V, n = n0 + r;
            const bool in = n < end && c < D;
            const T* src = in ? p + keys.key(n) * v.s + c : reinterpret_cast<const T*>(v.p);
            const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(dst + (r * S::LD + c) * sizeof(T)));
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(in ? 16 : 0) : "memory");
        }
    } else {
        for (int i = threadIdx.x; i < S::KT * DP; i += kThreads) {
            const int r = i / DP, c = i % DP, n = n0 + r;
            T x;
            heads::from_f(0.0f, x);
            if (n < end && c < D) x = p[keys.key(n) * v.s + c];
            reinterpret_cast<T*>(dst)[r * S::LD + c] = x;
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}

// Row r of a kv head's Sq * G: query r / G, head r % G of the group.
template <typename T, int DP, int RT>
__global__ void __launch_bounds__(kThreads) k_attention_few(const __grid_constant__ Problem p, Parts parts, int row_tiles, bool vec) {
    using S = Shape<T, DP, RT>;
    extern __shared__ __align__(16) unsigned char smem[];
    unsigned char *sk = smem, *sv = smem + 2 * S::TILE;
    constexpr int KT = S::KT;
    float *sq = reinterpret_cast<float*>(smem + 4 * S::TILE), *sp = sq + RT * DP, *sm = sp + RT * KT, *sl = sm + RT, *sf = sl + RT;
    pdl_begin();
    const int part = blockIdx.x % parts.parts, group = blockIdx.x / parts.parts;
    const int rt = group % row_tiles, hk = group / row_tiles % p.Hk, b = group / row_tiles / p.Hk;
    const Seq seq(p, b);
    const int off = seq.nk - seq.nq, R = p.Sq * p.G, r0 = rt * RT;
    const int first = r0 / p.G, last = (min(r0 + RT, R) - 1) / p.G;  // queries of the rows
    const Keys keys(p, seq.nk, first + off, min(last, seq.nq - 1) + off);
    const int all = first < seq.nq ? keys.count() : 0;
    const int share = (all + parts.parts - 1) / parts.parts;
    const int n0 = min(part * share, all), n1 = min(n0 + share, all);
    const int64_t ak = b * p.k.b + hk * p.k.h, av = b * p.v.b + hk * p.v.h;
    if (n0 < n1) {
        load_keys<T, DP, RT>(sk, p.k, ak, keys, n0, n1, p.D, vec);
        load_keys<T, DP, RT>(sv, p.v, av, keys, n0, n1, p.D, vec);
    }
    const float c = p.scale * kLog2e;
    for (int i = threadIdx.x; i < RT * DP; i += kThreads) {
        const int r = r0 + i / DP, col = i % DP;
        const bool in = r < R && r / p.G < seq.nq && col < p.D;
        sq[i] = in ? heads::to_f(reinterpret_cast<const T*>(p.q.p)[b * p.q.b + r / p.G * p.q.s + (hk * p.G + r % p.G) * p.q.h + col]) : 0.0f;
    }
    if (threadIdx.x < RT) sm[threadIdx.x] = -INFINITY, sl[threadIdx.x] = 0.0f;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // scores: a key and RH of the rows a thread
    constexpr int RH = RT * KT / kThreads;
    const int key = threadIdx.x % KT, half = threadIdx.x / KT;
    // sums: four columns (and those DP / 2 on, with 256) and a quarter of the rows
    constexpr int RQ = (RT + 3) / 4, NC = DP / 4 > 32 ? DP / 128 : 1, LANES = DP / 4 < 32 ? DP / 4 : 32;
    P2 acc[RQ][NC][2];
#pragma unroll
    for (auto& x : acc)
#pragma unroll
        for (auto& y : x) y[0] = y[1] = pack(0.0f, 0.0f);
    int stage = 0;
    for (int n = n0; n < n1; n += KT, stage ^= 1) {
        if (n + KT < n1) {
            load_keys<T, DP, RT>(sk + (stage ^ 1) * S::TILE, p.k, ak, keys, n + KT, n1, p.D, vec);
            load_keys<T, DP, RT>(sv + (stage ^ 1) * S::TILE, p.v, av, keys, n + KT, n1, p.D, vec);
            asm volatile("cp.async.wait_group 2;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();
        {
            const T* k = reinterpret_cast<const T*>(sk + stage * S::TILE) + key * S::LD;
            P2 s[RH];
#pragma unroll
            for (int i = 0; i < RH; ++i) s[i] = pack(0.0f, 0.0f);
#pragma unroll 2
            for (int d = 0; d < DP; d += S::V) {
                const heads::Pack<T, S::V> x = *reinterpret_cast<const heads::Pack<T, S::V>*>(k + d);
                P2 y[S::V / 2];
#pragma unroll
                for (int e = 0; e < S::V / 2; ++e) y[e] = pack(heads::to_f(x.v[2 * e]), heads::to_f(x.v[2 * e + 1]));
#pragma unroll
                for (int i = 0; i < RH; ++i)
#pragma unroll
                    for (int e = 0; e < S::V / 4; ++e) {
                        const float4 q = *reinterpret_cast<const float4*>(sq + (half * RH + i) * DP + d + 4 * e);
                        s[i] = fma2(pack(q.x, q.y), y[2 * e], s[i]);
                        s[i] = fma2(pack(q.z, q.w), y[2 * e + 1], s[i]);
                    }
            }
            const int j = n + key < n1 ? keys.key(n + key) : INT32_MAX;
#pragma unroll
            for (int i = 0; i < RH; ++i) {
                const int r = half * RH + i, q = (r0 + r) / p.G;
                const bool seen = q < seq.nq && r0 + r < R && q + off < seq.nk && sees(p, q + off, j);
                sp[r * KT + key] = seen ? sum2(s[i]) * c : -INFINITY;
            }
        }
        __syncthreads();
        // a warp takes every fourth row's maximum and sum
        for (int r = warp; r < RT; r += 4) {
            constexpr int N = KT / 32;
            float x[N], most = -INFINITY;
#pragma unroll
            for (int i = 0; i < N; ++i) most = fmaxf(most, x[i] = sp[r * KT + lane + 32 * i]);
#pragma unroll
            for (int m = 16; m >= 1; m >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, m));
            const float old = sm[r], now = fmaxf(old, most), ref = now == -INFINITY ? 0.0f : now;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x[i] = exp2f(x[i] - ref);
                sp[r * KT + lane + 32 * i] = x[i];
                sum += x[i];
            }
#pragma unroll
            for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
            __syncwarp();
            if (lane == 0) {
                const float f = exp2f(old - ref);
                sf[r] = f;
                sm[r] = now;
                sl[r] = fmaf(sl[r], f, sum);
            }
        }
        __syncthreads();
        if (lane < LANES) {
            const T* v = reinterpret_cast<const T*>(sv + stage * S::TILE);
#pragma unroll
            for (int i = 0; i < RQ; ++i) {
                const int r = warp * RQ + i;
                const P2 f = both(r < RT ? sf[r] : 0.0f);
#pragma unroll
                for (auto& y : acc[i]) y[0] = mul2(y[0], f), y[1] = mul2(y[1], f);
            }
#pragma unroll 2
            for (int k = 0; k < KT; k += 4) {
                float w[RQ][4];
#pragma unroll
                for (int i = 0; i < RQ; ++i)
                    *reinterpret_cast<float4*>(w[i]) =
                        warp * RQ + i < RT ? *reinterpret_cast<const float4*>(sp + (warp * RQ + i) * KT + k) : make_float4(0, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int m = 0; m < NC; ++m) {
                        const heads::Pack<T, 4> x = *reinterpret_cast<const heads::Pack<T, 4>*>(v + (k + e) * S::LD + 4 * lane + 128 * m);
                        const P2 y0 = pack(heads::to_f(x.v[0]), heads::to_f(x.v[1])), y1 = pack(heads::to_f(x.v[2]), heads::to_f(x.v[3]));
#pragma unroll
                        for (int i = 0; i < RQ; ++i) {
                            const P2 ww = both(w[i][e]);
                            acc[i][m][0] = fma2(ww, y0, acc[i][m][0]);
                            acc[i][m][1] = fma2(ww, y1, acc[i][m][1]);
                        }
                    }
            }
        }
        __syncthreads();
    }
    __syncthreads();
    if (lane >= LANES) return;
#pragma unroll
    for (int i = 0; i < RQ; ++i) {
        const int r = warp * RQ + i;
        if (r >= RT || r0 + r >= R) continue;
        const int q = (r0 + r) / p.G, h = hk * p.G + (r0 + r) % p.G;
        const int64_t row = (static_cast<int64_t>(b) * p.Hq + h) * p.Sq + q;
        const float l = sl[r];
        const bool any = l > 0.0f || isnan(l), whole = parts.parts == 1;
        const float f = whole ? (any ? 1.0f / l : 0.0f) : 1.0f;
#pragma unroll
        for (int m = 0; m < NC; ++m) {
            const float2 a = unpack(acc[i][m][0]), d = unpack(acc[i][m][1]);
            const float y[4] = {a.x * f, a.y * f, d.x * f, d.y * f};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = 4 * lane + 128 * m + e;
                if (col >= p.D) continue;
                if (whole)
                    heads::from_f(y[e], reinterpret_cast<T*>(p.o.p)[b * p.o.b + q * p.o.s + h * p.o.h + col]);
                else
                    parts.sum[(row * parts.parts + part) * p.D + col] = y[e];
            }
        }
        if (lane == 0) {
            if (!whole) {
                parts.stat[(row * parts.parts + part) * 2] = sm[r];
                parts.stat[(row * parts.parts + part) * 2 + 1] = l;
            } else if (p.lse) {
                p.lse[row] = any ? (sm[r] + log2f(l)) * kLn2 : -INFINITY;
            }
        }
    }
}

// The parts of a row joined in a fixed order: by a warp, or by eight with every eighth part each where
// there are more than eight parts or few rows.
constexpr int kMaxParts = 128, kJoinWarps = 8;
template <typename T> __global__ void __launch_bounds__(32 * kJoinWarps) k_attention_join(const __grid_constant__ Problem p, Parts parts, int64_t rows, int per_row) {
    __shared__ float weight[kJoinWarps][kMaxParts], part[kJoinWarps][256];
    pdl_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp & (per_row - 1);
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kJoinWarps / per_row) + warp / per_row;
    if (row >= rows) return;  // with eight warps a row, all or none of the CTA
    const int q = static_cast<int>(row % p.Sq), h = static_cast<int>(row / p.Sq % p.Hq), b = static_cast<int>(row / p.Sq / p.Hq);
    const float* sum = parts.sum + row * parts.parts * p.D;
    float m[kMaxParts / 32], l[kMaxParts / 32], top = -INFINITY, norm = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxParts / 32; ++i) {
        const int k = lane + 32 * i;
        const float2 st = k < parts.parts ? reinterpret_cast<const float2*>(parts.stat)[row * parts.parts + k] : make_float2(-INFINITY, 0.0f);
        m[i] = st.x;
        l[i] = st.y;
        top = fmaxf(top, st.x);
    }
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < kMaxParts / 32; ++i) {
        const float f = exp2f(m[i] - ref);
        weight[warp][lane + 32 * i] = f;
        norm = fmaf(l[i], f, norm);
    }
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) norm += __shfl_xor_sync(0xffffffffu, norm, k);
    __syncwarp();
    const bool any = norm > 0.0f || isnan(norm);
    const float f = any ? 1.0f / norm : 0.0f;
    T* o = reinterpret_cast<T*>(p.o.p) + b * p.o.b + q * p.o.s + h * p.o.h;
    float acc[8] = {};  // columns lane + 32 j
#pragma unroll 4
    for (int i = sub; i < parts.parts; i += per_row)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (lane + 32 * j < p.D) acc[j] = fmaf(sum[static_cast<int64_t>(i) * p.D + lane + 32 * j], weight[warp][i], acc[j]);
    if (per_row == 1) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (lane + 32 * j < p.D) heads::from_f(acc[j] * f, o[lane + 32 * j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) part[warp][lane + 32 * j] = acc[j];
        __syncthreads();
        for (int c = threadIdx.x; c < p.D; c += 32 * kJoinWarps) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < kJoinWarps; ++i) s += part[i][c];
            heads::from_f(s * f, o[c]);
        }
    }
    if (p.lse && sub == 0 && lane == 0) p.lse[row] = any ? (top + log2f(norm)) * kLn2 : -INFINITY;
}

template <typename T, int DP, int RT> qsml_status_t run(Context* ctx, const Problem& p, bool vec) {
    using S = Shape<T, DP, RT>;
    const auto kernel = k_attention_few<T, DP, RT>;
    const char* name = "k_attention_few";
    QSML_TRY_STATUS(check_cuda(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::SMEM)), name));
    int resident = 1;
    QSML_TRY_STATUS(check_cuda(ctx, cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, kThreads, S::SMEM), name));
    const int R = p.Sq * p.G, row_tiles = (R + RT - 1) / RT;
    const int64_t groups = static_cast<int64_t>(row_tiles) * p.Hk * p.B;
    const int64_t n = few_parts(ctx, p, groups, std::max(resident, 1), 2 * S::KT, INT64_MAX);
    if (groups * n > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "qsml_attention: dimensions too large");
    Workspace ws(ctx);
    Parts parts;
    QSML_TRY_STATUS(get_parts(ctx, &ws, p, n, &parts));
    const cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(groups * parts.parts)), dim3(kThreads), S::SMEM, ctx->stream, p, parts, row_tiles, vec);
    if (e != cudaSuccess) return check_cuda(ctx, e, name);
    QSML_TRY_STATUS(after_launch(ctx, name));
    return join_parts(ctx, p, parts);
}

template <typename T> qsml_status_t forward(Context* ctx, const Problem& p) {
    const int64_t es = sizeof(T);
    const bool vec = p.D * es % 16 == 0 && heads::rows_on(p.k, es, 16) && heads::rows_on(p.v, es, 16);
    const int R = p.Sq * p.G;
    return by_width(p.D, [&](auto width) {
        constexpr int DP = decltype(width)::value;
        if (R <= 4) return run<T, DP, 4>(ctx, p, vec);
        if (R <= 8 || (sizeof(T) == 4 && DP == 256)) return run<T, DP, 8>(ctx, p, vec);
        if constexpr (sizeof(T) == 4 && DP == 256)
            return static_cast<qsml_status_t>(QSML_E_UNSUPPORTED);
        else
            return run<T, DP, 16>(ctx, p, vec);
    });
}

}  // namespace

// Up to 16 rows a kv head, and up to 64 over many keys, which more CTAs then share (64 queries of one head
// over themselves take 19 us here, 7 by tiles).
bool few_queries(const Problem& p) {
    const int64_t rows = static_cast<int64_t>(p.Sq) * p.G;
    return rows <= 16 || (rows <= 64 && p.Sk >= 4 * rows);
}

int64_t few_parts(Context* ctx, const Problem& p, int64_t groups, int resident, int least, int64_t longest) {
    // no row sees more keys than these
    const int64_t visible = p.window ? std::min<int64_t>(p.Sk, static_cast<int64_t>(p.window) + p.sinks + p.Sq) : p.Sk;
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kMaxParts, (visible + least - 1) / least));
    // The time of n parts: waves of CTAs (whole ones, where all are alike), each of a part's keys and
    // of what a CTA takes besides, as long as START keys (128, 256, 512 and 1024 measured, each call on keys out of
    // L2: binary16 of 8 heads of 128, 16 sequences over 1 to 8192 keys 69, 67, 73, 73 us; 8 over 1 to 16384 62, 59, 57,
    // 64; 64 over 1 to 2048 71, 71, 71, 65; 64 over 2048 of 16 heads of 64 102, 102, 90, 90; binary32, 5 over 1 to
    // 8192 of 8 heads of 64 54, 56, 50, 67; one sequence, and 4 over 4096, the same with each).
    constexpr double START = 512.0;
    const double slots = static_cast<double>(ctx->num_sms) * resident;
    const int64_t fewest = std::max<int64_t>(1, std::min<int64_t>(most, visible / longest + (visible % longest != 0)));
    int64_t best = fewest;
    double least_time = 0.0;
    for (int64_t n = fewest; n <= most; ++n) {
        const double waves = static_cast<double>(groups * n) / slots;
        const double time = (p.nk ? waves + 1.0 : std::ceil(waves)) * (static_cast<double>(visible) / n + START);
        if (n == fewest || time < least_time) best = n, least_time = time;
    }
    return best;
}

qsml_status_t get_parts(Context* ctx, Workspace* ws, const Problem& p, int64_t n, Parts* out) {
    out->parts = static_cast<int>(n);
    if (n == 1) return QSML_OK;
    const int64_t rows = static_cast<int64_t>(p.B) * p.Hq * p.Sq;
    void* m = nullptr;
    // the pairs of statistics first, so that they lie on 8 bytes and the sums on 16 whatever rows * n * D is
    const int64_t stats = (rows * n * 2 + 3) / 4 * 4;
    QSML_TRY_STATUS(ws->get(sizeof(float) * (stats + rows * n * p.D), &m));
    out->stat = static_cast<float*>(m);
    out->sum = out->stat + stats;
    return QSML_OK;
}

qsml_status_t join_parts(Context* ctx, const Problem& p, const Parts& parts) {
    if (parts.parts == 1) return QSML_OK;
    const int64_t rows = static_cast<int64_t>(p.B) * p.Hq * p.Sq;
    if (rows > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "qsml_attention: dimensions too large");
    const int per_row = parts.parts > kJoinWarps || rows <= 4096 ? kJoinWarps : 1, at_once = kJoinWarps / per_row;
    const cudaError_t e = launch_pdl(p.f16 ? k_attention_join<__half> : k_attention_join<float>, dim3(static_cast<unsigned>((rows + at_once - 1) / at_once)),
                                     dim3(32 * kJoinWarps), 0, ctx->stream, p, parts, rows, per_row);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_attention_join");
    return after_launch(ctx, "k_attention_join");
}

qsml_status_t forward_few(Context* ctx, const Problem& p) {
    if (few_tc_takes(p)) return forward_few_tc(ctx, p);
    return p.f16 ? forward<__half>(ctx, p) : forward<float>(ctx, p);
}

}  // namespace attn
}  // namespace qsml
