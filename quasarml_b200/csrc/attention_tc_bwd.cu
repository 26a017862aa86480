// Attention's gradients on the tensor cores (binary16, heads of up to 128 columns).
//
// With P = exp(scale q k^T - lse), dP = dout v^T, dS = P (dP - delta):
//   dq = scale dS k,   dk = scale dS^T q,   dv = P^T dout.
// k_attention_prepare takes delta = sum(dout o) of each row, lse in base 2, and the largest
// |dout|, |o| and |v| of each head.  k_attention_dq goes over a tile of queries' keys, k_attention_dkv over
// the queries of all heads of the group that see a tile of keys: P and dP are computed in both,
// seven products instead of five, and no sum is shared between CTAs.  The accumulators stay in
// TMEM (dkv: S^T, dP^T, dV and dK of 128 columns fill it); P^T and dS^T (dq: dS) are left there
// as binary16 by the threads that compute them, a row and half of its columns each, and are the
// next products' A operand.  While they work on one product the tensor core does the next.
// Bound by the tensor core and the exponentials in turn: of a tile of 128 x 128 with 128
// columns, 2048 (dkv) and 1536 (dq) cycles of products, and 1024 of exponentials.
// dS is rounded to binary16 between two products.  It is computed times a power of two that
// brings 2 |dout| |v|, which bounds it, to [2^14, 2^15], and which the sums are divided by: in dq that of
// the head, in dkv that of the largest head of the group, whose terms share a sum.  Only rows that take part
// and are finite count, so that no sequence or kv head costs another bits.
// A row whose keys are all in one tile takes delta = sum(P dP) instead of sum(dout o): with a few
// keys the rounding of o would be the largest error of dq and dk (alone 0.00033 of their norm, where
// their own rounding is 0.00021).  Measured, 2 x 4096 tokens of 16 heads over 2 with 128 columns, window
// 2048: 424 us in short runs, dkv 241 (a step 3560 cycles) and dq 184 (2600); 467 back to back, under the power
// cap.  With 128 columns both kernels reload spilled registers, dq 248 bytes and dkv 108.
#include <algorithm>

#include "attention_tc.cuh"

namespace qsml {
namespace attn {
namespace {

constexpr int kThreads = 384, FEW = 56, MANY = 224;  // registers of the control warpgroup and the two others, of 3 x 168

// P is computed times 2^14, so that weights down to 2^-28 are normal numbers of binary16.
constexpr float SHIFT = 14.0f;

struct Stats {
    float *minus, *delta;  // [B * Hq, pitch]; minus: SHIFT - lse in base 2, -inf where a row sees nothing
    unsigned *of_q, *of_v;  // bits of the largest squared norms: [B * Hq][2] of dout's and o's rows, [B * Hk] of v's
    int64_t pitch;
};

// A CTA takes 128 rows of a head (blocks below qblocks: of dout and o, then of v), 16 lanes a row.
__global__ void __launch_bounds__(256, 4) k_attention_prepare(const __grid_constant__ Problem p, Stats st, int qblocks) {
    pdl_begin();
    const int lane = threadIdx.x & 15, row = threadIdx.x >> 4;
    const bool of_q = static_cast<int>(blockIdx.x) < qblocks;
    const int i = of_q ? blockIdx.x : blockIdx.x - qblocks, H = of_q ? p.Hq : p.Hk;
    const int bh = i % (p.B * H), first = i / (p.B * H) * TILE, b = bh / H, h = bh - b * H;
    const Seq seq(p, b);
    const int n = of_q ? seq.nq : seq.nk, off = seq.nk - seq.nq;
    // rows that take part: queries that see a key, keys that a query sees
    const Keys keys(p, seq.nk, off, seq.nk - 1);
    const int from = of_q ? -off : keys.lo, sink = of_q ? 0 : keys.sink;
    const bool mine = lane * 8 < p.D;
    auto at = [&](const View& v, int r) { return reinterpret_cast<const uint4*>(reinterpret_cast<const __half*>(v.p) + b * v.b + h * v.h + r * v.s + lane * 8); };
    auto sum = [&](const uint4& x, const uint4& y) {
        const __half2 *u = reinterpret_cast<const __half2*>(&x), *w = reinterpret_cast<const __half2*>(&y);
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = __half22float2(u[e]), g = __half22float2(w[e]);
            s = fmaf(f.x, g.x, fmaf(f.y, g.y, s));
        }
#pragma unroll
        for (int m = 8; m >= 1; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        return s;
    };
    float most[2] = {0.0f, 0.0f};
    auto larger = [](float m, float x) { return x < INFINITY ? fmaxf(m, x) : m; };  // of numbers
    constexpr int ROWS = 4;  // of a lane at once: with all eight two CTAs fit a SM, and their waves took 30 us
    for (int r0 = first + row; r0 < first + TILE; r0 += 16 * ROWS) {
        uint4 x[ROWS], y[ROWS];
        float lse[ROWS];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            const int r = r0 + 16 * k;
            lse[k] = of_q && lane == 0 && r < n ? p.lse[static_cast<int64_t>(bh) * p.Sq + r] : -INFINITY;
            x[k] = y[k] = make_uint4(0, 0, 0, 0);
            if (r < n && mine) {
                x[k] = *at(of_q ? p.dout : p.v, r);
                if (of_q) y[k] = *at(p.o, r);
            }
        }
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            const int r = r0 + 16 * k;
            const bool takes_part = r >= from || r < sink;
            const float xx = sum(x[k], x[k]);
            if (takes_part) most[0] = larger(most[0], xx);
            if (!of_q) continue;
            const float yy = sum(y[k], y[k]);
            if (takes_part) most[1] = larger(most[1], yy);
            const float delta = sum(x[k], y[k]);
            if (lane == 0) {
                st.minus[bh * st.pitch + r] = lse[k] == -INFINITY ? -INFINITY : fmaf(lse[k], -kLog2e, SHIFT);
                st.delta[bh * st.pitch + r] = delta;
            }
        }
    }
    // one atomic a CTA
    __shared__ float largest[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float m = most[k];
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        if ((threadIdx.x & 31) == 0) largest[k][threadIdx.x >> 5] = m;
    }
    __syncthreads();
    if (threadIdx.x < (of_q ? 2 : 1)) {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, largest[threadIdx.x][i]);
        // bits of numbers that are not negative are in their order; the largest does not depend on it
        if (m > 0.0f) atomicMax(of_q ? st.of_q + 2 * static_cast<int64_t>(bh) + threadIdx.x : st.of_v + bh, __float_as_uint(m));
    }
}

// The power of two that the dS of n query heads (of all sequences' heads) of a kv head is multiplied by: 2^15 at
// most after it.
__device__ __forceinline__ float gain_of(const Stats& st, int head, int n, int kv_head) {
    float g = 0.0f, o = 0.0f;
    const float v = __uint_as_float(st.of_v[kv_head]);
#pragma unroll 4
    for (int i = head; i < head + n; ++i) {
        const uint2 m = reinterpret_cast<const uint2*>(st.of_q)[i];
        g = fmaxf(g, __uint_as_float(m.x));
        o = fmaxf(o, __uint_as_float(m.y));
    }
    const float bound = sqrtf(g) * (sqrtf(o) + sqrtf(v));
    if (!(bound > 0.0f && bound < INFINITY)) return 1.0f;
    int e;
    frexpf(bound, &e);  // bound < 2^e
    return exp2f(static_cast<float>(min(max(15 - e, -100), 100)));
}

// Registers of 64 columns of scores to 2^SHIFT P = 2^(s c + minus), minus(e) of columns 2 e and 2 e + 1;
// the exponents of a pair in turn with the exponentials of one before.
template <typename L> __device__ __forceinline__ void weights(uint32_t (&r)[64], float c, L&& minus) {
    const P2 c2 = both(c);
    constexpr int AHEAD = 4;
#pragma unroll
    for (int e = 0; e < 32 + AHEAD; ++e) {
        if (e < 32) {
            const float2 x = unpack(fma2(pack(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), c2, minus(e)));
            r[2 * e] = __float_as_uint(x.x);
            r[2 * e + 1] = __float_as_uint(x.y);
        }
        if (e >= AHEAD) {
            const int k = 2 * (e - AHEAD);
            r[k] = __float_as_uint(exp2_fast(__uint_as_float(r[k])));
            r[k + 1] = __float_as_uint(exp2_fast(__uint_as_float(r[k + 1])));
        }
    }
}
// 64 columns of this thread's lane.
__device__ __forceinline__ void load64(uint32_t at, uint32_t (&r)[64]) {
    tmem_ld32_start(at, r);
    tmem_ld32_start(at + 32, r + 32);
    tmem_wait(r);
    tmem_wait(r + 32);
}
__device__ __forceinline__ void keep(uint32_t (&r)[64], uint32_t lo, uint32_t hi) {
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        r[e] = lo & (1u << e) ? r[e] : 0xff800000u;
        r[32 + e] = hi & (1u << e) ? r[32 + e] : 0xff800000u;
    }
}
// Half of a row's binary16 in place, then the arrival of its warp.
__device__ __forceinline__ void arrive(uint32_t bar) {
    tmem_st_wait();
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// A row of sums in TMEM (none: zeros), with what is kept of it (null: nothing), times f, as binary32.
template <int DP> __device__ __forceinline__ void store_sums(uint32_t at, bool any, float f, float* to, int D, const float* kept) {
#pragma unroll
    for (int c = 0; c < DP; c += 32) {
        if (c >= D) break;
        uint32_t r[32];
        if (any) load_sums(at + c, r, kept ? kept + c * TILE : nullptr, D - c, 1.0f);
#pragma unroll
        for (int j = 0; j < 32; j += 4)
            if (c + j < D)
                *reinterpret_cast<float4*>(to + c + j) =
                    any ? make_float4(__uint_as_float(r[j]) * f, __uint_as_float(r[j + 1]) * f, __uint_as_float(r[j + 2]) * f, __uint_as_float(r[j + 3]) * f)
                        : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
}

struct BwdMaps {
    HeadMap q, k, v, g;
};

// The steps of a tile of keys (tiles of queries that see it, of all heads of the group) over several
// CTAs: the tiles with sinks, which all later queries see, in `many` parts, the others in `few`.  A
// part's dk and dv are binary32 tiles [128][D] each in `sum`, where its tile has more than one; a part of
// more than DRAIN steps keeps its sums in tiles of `kept` on the way.
struct KeyParts {
    float *sum, *kept;
    int many, few, sink_tiles, tiles;
    __host__ __device__ int64_t slots() const { return static_cast<int64_t>(sink_tiles) * many + static_cast<int64_t>(tiles - sink_tiles) * few; }
    __host__ __device__ int64_t slot(int tile) const {
        return tile < sink_tiles ? static_cast<int64_t>(tile) * many
                                 : static_cast<int64_t>(sink_tiles) * many + static_cast<int64_t>(tile - sink_tiles) * few;
    }
    __host__ __device__ int parts(int tile) const { return tile < sink_tiles ? many : few; }
};

template <int DP> struct Dkv {
    static constexpr int STAGE = 2 * TileOf<DP>::BYTES;
    static constexpr size_t SMEM = 2 * size_t(TileOf<DP>::BYTES) + 2 * (STAGE + 1024) + 1024 + 8 * 16 + 16;
};

template <int DP, bool LONG>
__global__ void __launch_bounds__(kThreads, 1)
    k_attention_dkv(const __grid_constant__ Problem p, const __grid_constant__ BwdMaps maps, Stats st, KeyParts kp, int* status) {
    using L = Dkv<DP>;
    constexpr int BYTES = TileOf<DP>::BYTES;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    const uint32_t k_tile = base, v_tile = base + BYTES;
    auto q_tile = [&](int s) { return base + 2 * BYTES + s * L::STAGE; };
    auto g_tile = [&](int s) { return q_tile(s) + BYTES; };
    const uint32_t stat = base + 2 * BYTES + 2 * L::STAGE;  // a stage's minus and delta
    const float* stats = reinterpret_cast<const float*>(smem_raw + (stat - raw));
    const uint32_t bars = stat + 2 * 1024;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 16 + 8u * s; };
    const uint32_t kv_full = bars + 32, land = bars + 40, drain = bars + 48, sums_full = bars + 56, s_full = bars + 64, dp_full = bars + 72;
    auto p_ready = [&](int w) { return bars + 80 + 8u * w; };
    auto ds_ready = [&](int w) { return bars + 96 + 8u * w; };
    unsigned char* misc = smem_raw + (bars - raw) + 128;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
            mbar_init(p_ready(s), 4);
            mbar_init(ds_ready(s), 4);
        }
        for (uint32_t b = kv_full; b <= dp_full; b += 8) mbar_init(b, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;  // S^T and P^T, dP^T and dS^T, dV, dK
    pdl_begin();
    const long long limit = wait_limit(status);

    // the first keys, which the most queries see, first
    const int hk = blockIdx.x % p.Hk, b = blockIdx.x / p.Hk % p.B, slot = blockIdx.x / p.Hk / p.B;
    const int rest = slot - kp.sink_tiles * kp.many, tile = rest < 0 ? slot / kp.many : kp.sink_tiles + rest / kp.few;
    const int k0 = tile * TILE, parts = kp.parts(tile), part = slot - static_cast<int>(kp.slot(tile));
    const Seq seq(p, b);
    const int off = seq.nk - seq.nq;
    const Queries qs(p, seq, k0, k0 + TILE);
    const int t0 = qs.lo / TILE, per = qs.hi > qs.lo ? (qs.hi + TILE - 1) / TILE - t0 : 0;  // tiles of queries a head
    const int share = (per * p.G + parts - 1) / parts, step0 = min(part * share, per * p.G), steps = min(share, per * p.G - step0);
    auto fresh = [](int n) { return LONG ? n % DRAIN == 0 : n == 0; };  // whether the sums begin with step n

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FEW));
        if (warp == 0 && steps > 0) {
            const bool issue = elect_one();
            bool ok = true, land_open = false;
            uint32_t land_phase = 0;
            int flying[2] = {-1, -1};  // phase of a stage's last load that has no other wait
            if (issue) {
                mbar_expect_tx(kv_full, 2 * BYTES);
                load_tile<DP>(k_tile, maps.k, kv_full, k0, hk, b);
                load_tile<DP>(v_tile, maps.v, kv_full, k0, hk, b);
            }
            for (int n = 0; n < steps && ok; ++n) {
                const int s = n & 1, h = hk * p.G + (step0 + n) / per, q0 = (t0 + (step0 + n) % per) * TILE;
                ok = warp_wait(empty(s), (n >> 1 & 1) ^ 1, abort_flag, limit);
                if (!ok) break;
                const bool ragged = q0 + TILE > seq.nq;
                const uint32_t bar = ragged ? land : full(s);
                if (issue) {
                    mbar_expect_tx(bar, L::STAGE + 1024);
                    load_tile<DP>(q_tile(s), maps.q, bar, q0, h, b);
                    load_tile<DP>(g_tile(s), maps.g, bar, q0, h, b);
                    const int64_t at = (static_cast<int64_t>(b) * p.Hq + h) * st.pitch + q0;
                    for (int i = 0; i < 2; ++i)
                        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                                     ::"r"(stat + s * 1024 + i * 512), "l"((i ? st.delta : st.minus) + at), "r"(512), "r"(bar) : "memory");
                }
                flying[s] = ragged ? -1 : n >> 1 & 1;
                if (!ragged) continue;
                ok = warp_wait(land, land_phase, abort_flag, limit);
                land_open = !ok;
                if (!ok) break;
                land_phase ^= 1u;
                clear_rows<DP>(q_tile(s), q0, 0, 0, seq.nq);
                clear_rows<DP>(g_tile(s), q0, 0, 0, seq.nq);
                if (issue) mbar_arrive(full(s));
            }
            const long long start = clock64();
            while (!mbar_test(kv_full, 0) && clock64() - start < WAIT_CYCLES) {
            }
            for (int s = 0; s < 2; ++s)
                while (flying[s] >= 0 && !mbar_test(full(s), static_cast<uint32_t>(flying[s])) && clock64() - start < WAIT_CYCLES) {
                }
            while (land_open && !mbar_test(land, land_phase) && clock64() - start < WAIT_CYCLES) {
            }
        } else if (warp == 1 && steps > 0) {
            const bool issue = elect_one();
            bool ok = warp_wait(kv_full, 0, abort_flag, limit);
            const uint64_t kd = score_desc(k_tile), vd = score_desc(v_tile);
            // x += a operand in two halves as they come, times a tile.  Where the sums begin anew, warpgroup 0 has
            // moved dV and warpgroup 1 dK before their P of the step was ready
            auto sums = [&](uint32_t d, uint32_t a, uint32_t tile, uint32_t bar, int n) {
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    if (!warp_wait(bar + 8 * w, n & 1, abort_flag, limit)) return false;
                    tc_fence_after();
                    mma_sums<DP, 64>(issue, d, a + 64 * w, desc_on(sum_desc<DP>(tile), w * 64 * 128), !fresh(n) || w > 0);
                }
                return true;
            };
            // what is left in S^T and dP^T has been read when the next is written, MMAs being executed
            // in the order of their issue
            auto begin = [&](int n, bool second) {
                const int s = n & 1;
                if (!second && !warp_wait(full(s), n >> 1 & 1, abort_flag, limit)) return false;
                tc_fence_after();
                mma_scores<DP, TILE>(issue, tmem + (second ? TILE : 0), second ? vd : kd, score_desc(second ? g_tile(s) : q_tile(s)));
                if (issue) mma_commit(second ? dp_full : s_full);
                return true;
            };
            ok = ok && begin(0, false) && begin(0, true);
            for (int n = 0; n < steps && ok; ++n) {
                ok = sums(tmem + 256, tmem, g_tile(n & 1), p_ready(0), n);
                if (ok && n + 1 < steps) ok = begin(n + 1, false);
                ok = ok && sums(tmem + 256 + DP, tmem + TILE, q_tile(n & 1), ds_ready(0), n);
                if (!ok) break;
                if (issue) mma_commit(empty(n & 1));
                if (n + 1 < steps) ok = begin(n + 1, true);
            }
            if (ok && issue) mma_commit(sums_full);
            if (issue) mma_commit(drain);
            const long long start = clock64();
            while (!mbar_test(drain, 0) && clock64() - start < WAIT_CYCLES) {
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(MANY));
        const int w = (warp - 4) >> 2, quarter = warp & 3, k = k0 + quarter * 32 + lane;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        const uint32_t s_at = lanes + 64 * w, dp_at = lanes + TILE + 64 * w;
        const float c = p.scale * kLog2e, gain = gain_of(st, b * p.Hq + hk * p.G, p.G, b * p.Hk + hk), ds_gain = gain * exp2f(-SHIFT);
        const int last_key = min(k0 + TILE, seq.nk) - 1;
        // a warpgroup each: dV and dK
        const View& to = w ? p.dk : p.dv;
        const uint32_t sums_at = lanes + 256 + w * DP;
        const int64_t out_tile = (((static_cast<int64_t>(slot) * p.B + b) * p.Hk + hk) * 2 + w) * TILE * p.D;
        auto kept_row = [&] { return kept_at(kp.kept + out_tile, k - k0, 0); };
        bool ok = true;
        for (int n = 0; n < steps && ok; ++n) {
            const int s = n & 1, q0 = (t0 + (step0 + n) % per) * TILE;
            const float *minus = stats + s * 256 + 64 * w, *delta = minus + 128;
            ok = warp_wait(s_full, n & 1, abort_flag, limit) && warp_wait(full(s), n >> 1 & 1, abort_flag, limit);
            if (LONG && ok && n > 0 && fresh(n)) {  // dP^T comes after all sums of the step before
                ok = warp_wait(dp_full, n & 1, abort_flag, limit);
                if (!ok) break;
                tc_fence_after();
                keep_sums<DP>(sums_at, kept_row(), p.D, n == DRAIN, 1.0f);
            }
            if (!ok) break;
            tc_fence_after();
            uint32_t r[64];
            load64(s_at, r);
            // queries at positions from k on, and before k + window
            const int pos = q0 + off;
            if (pos < last_key || (p.window && pos + TILE - 1 - k0 >= p.window && k0 + TILE > p.sinks)) {
                const int lo = k - pos - 64 * w, hi = p.window && k >= p.sinks ? lo + p.window : 64;
                keep(r, below(hi) & ~below(lo), below(hi - 32) & ~below(lo - 32));
            }
            weights(r, c, [&](int e) {
                const float2 l = *reinterpret_cast<const float2*>(minus + 2 * e);
                return pack(l.x, l.y);
            });
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t f[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) f[e] = half2_of(__uint_as_float(r[32 * h + 2 * e]), __uint_as_float(r[32 * h + 2 * e + 1]));
                tmem_st16(s_at + 16 * h, f);
            }
            arrive(p_ready(w));
            if (sees_one(p, pos + TILE) || (pos <= 0 && pos > -TILE)) {  // queries whose dS is 0: all, or that at position 0
#pragma unroll
                for (int e = 0; e < 64; ++e)
                    if (sees_one(p, pos + 64 * w + e)) r[e] = 0;
            }
            ok = warp_wait(dp_full, n & 1, abort_flag, limit);
            if (!ok) break;
            tc_fence_after();
            uint32_t d[64];
            load64(dp_at, d);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t f[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int i = 32 * h + 2 * e;
                    const float2 l = *reinterpret_cast<const float2*>(delta + i);
                    const P2 x = sub2(pack(__uint_as_float(d[i]), __uint_as_float(d[i + 1])), pack(l.x, l.y));
                    const float2 y = unpack(mul2(mul2(pack(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), both(ds_gain)), x));
                    f[e] = half2_of(y.x, y.y);
                }
                tmem_st16(dp_at + 16 * h, f);
            }
            arrive(ds_ready(w));
        }
        if (ok && steps > 0) ok = warp_wait(sums_full, 0, abort_flag, limit);
        tc_fence_after();
        const float* prior = LONG && steps > DRAIN ? kept_row() : nullptr;
        const float f = w ? p.scale / gain : exp2f(-SHIFT);
        if (ok && parts > 1) {
            store_sums<DP>(sums_at, steps > 0, f, kp.sum + out_tile + static_cast<int64_t>(k - k0) * p.D, p.D, prior);
        } else if (ok && to.p) {
            __half* row = k < p.Sk ? reinterpret_cast<__half*>(to.p) + b * to.b + k * to.s + hk * to.h : nullptr;
            if (steps > 0) {
                const bool live = k < seq.nk;
                store_row<DP>(sums_at, f, live ? row : nullptr, p.D, prior);
                if (row && !live) zero_row(row, p.D);
            } else if (row) {
                zero_row(row, p.D);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag && threadIdx.x == 0) atomicExch(status, QSML_E_TIMEOUT);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// dk and dv of the tiles in several parts: the parts' sums, added in their order; a quarter of a tile a
// CTA, 8 columns a thread.
__global__ void __launch_bounds__(256) k_attention_dkv_join(const __grid_constant__ Problem p, KeyParts kp, int tiles) {
    pdl_begin();
    const int units = p.D / 8, w = blockIdx.y;
    const View& to = w ? p.dk : p.dv;
    const int quarter = blockIdx.x & 3, tile = (blockIdx.x >> 2) % tiles, bh = (blockIdx.x >> 2) / tiles, b = bh / p.Hk, hk = bh - b * p.Hk;
    const int parts = kp.parts(tile), nk = Seq(p, b).nk;
    const int64_t stride = static_cast<int64_t>(p.B) * p.Hk * 2 * TILE * p.D;
    const float* from = kp.sum + (kp.slot(tile) * p.B * p.Hk + bh) * 2 * TILE * p.D + static_cast<int64_t>(w) * TILE * p.D;
    if (!to.p || parts == 1) return;
    for (int i = threadIdx.x; i < TILE / 4 * units; i += 256) {
        const int row = i / units, r = quarter * (TILE / 4) + row, c = (i - row * units) * 8, k = tile * TILE + r;
        if (k >= p.Sk) break;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y = x;
        if (k < nk) {
#pragma unroll 4
            for (int n = 0; n < parts; ++n) {
                const float4* a = reinterpret_cast<const float4*>(from + n * stride + static_cast<int64_t>(r) * p.D + c);
                const float4 u = a[0], v = a[1];
                x.x += u.x, x.y += u.y, x.z += u.z, x.w += u.w;
                y.x += v.x, y.y += v.y, y.z += v.z, y.w += v.w;
            }
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<__half*>(to.p) + b * to.b + k * to.s + hk * to.h + c) =
            make_uint4(half2_of(x.x, x.y), half2_of(x.z, x.w), half2_of(y.x, y.y), half2_of(y.z, y.w));
    }
}

template <int DP> struct Dq {
    static constexpr int KS = 3, VS = 2;  // slots of K (read by S and dq) and V
    static constexpr size_t SMEM = (2 + KS + VS) * size_t(TileOf<DP>::BYTES) + 1024 + 8 * 24 + 16 + 1024;
    static_assert(SMEM <= 232448, "shared memory");
};

template <int DP, bool LONG>
__global__ void __launch_bounds__(kThreads, 1)
    k_attention_dq(const __grid_constant__ Problem p, const __grid_constant__ BwdMaps maps, Stats st, int tiles, float* kept, int* status) {
    using L = Dq<DP>;
    constexpr int BYTES = TileOf<DP>::BYTES;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    const uint32_t q_tile = base, g_tile = base + BYTES;
    auto slot = [&](int v, int n) { return base + (2 + (v ? L::KS + n % L::VS : n % L::KS)) * BYTES; };
    float* part = reinterpret_cast<float*>(smem_raw + (base - raw) + (2 + L::KS + L::VS) * BYTES);  // [2][128]
    const uint32_t bars = base + (2 + L::KS + L::VS) * BYTES + 1024;
    // K's slots, then V's
    auto full = [&](int v, int n) { return bars + 8u * (v ? L::KS + n % L::VS : n % L::KS); };
    auto empty = [&](int v, int n) { return full(v, n) + 8u * (L::KS + L::VS); };
    auto turn = [&](int v, int n) { return static_cast<uint32_t>(n / (v ? L::VS : L::KS)) & 1u; };
    const uint32_t q_full = bars + 80, land = bars + 88, drain = bars + 96, sums_full = bars + 104, dp_full = bars + 112;
    auto s_full = [&](int n) { return bars + 120 + 8u * (n & 1); };
    auto ds_ready = [&](int w) { return bars + 136 + 8u * w; };
    const uint32_t part_full = bars + 152;
    unsigned char* misc = smem_raw + (bars - raw) + 8 * 24;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (uint32_t b = bars; b < bars + 136; b += 8) mbar_init(b, 1);
        mbar_init(ds_ready(0), 4);
        mbar_init(ds_ready(1), 4);
        mbar_init(part_full, 8);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;  // S in two buffers, dP and dS, dQ
    pdl_begin();
    const long long limit = wait_limit(status);

    // the last queries of all sequences, with the most keys, first
    const int bh = blockIdx.x % (p.B * p.Hq), b = bh / p.Hq, h = bh - b * p.Hq, hk = h / p.G;
    const int q0 = (tiles - 1 - blockIdx.x / (p.B * p.Hq)) * TILE;
    const Seq seq(p, b);
    const int off = seq.nk - seq.nq;
    const Keys keys(p, seq.nk, q0 + off, min(q0 + TILE, seq.nq) - 1 + off);
    const Tiles list(keys, TILE);
    const int steps = q0 < seq.nq ? list.n : 0;
    auto fresh = [](int n) { return LONG ? n % DRAIN == 0 : n == 0; };  // whether dQ begins with step n

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FEW));
        if (warp == 0 && steps > 0) {
            const bool issue = elect_one();
            bool ok = true, land_open = false;
            uint32_t land_phase = 0;
            if (issue) {
                mbar_expect_tx(q_full, 2 * BYTES);
                load_tile<DP>(q_tile, maps.q, q_full, q0, h, b);
                load_tile<DP>(g_tile, maps.g, q_full, q0, h, b);
            }
            uint32_t flying = 0, parity = 0;  // by slot: whether its last load has no other wait, and its phase
            for (int n = 0; n < steps && ok; ++n) {
                const int k0 = list.tile(n) * TILE;
                const bool ragged = k0 + TILE > keys.hi || (k0 < keys.lo && k0 + TILE > keys.sink);
                for (int v = 0; v < 2; ++v) {
                    ok = warp_wait(empty(v, n), turn(v, n) ^ 1u, abort_flag, limit);
                    if (!ok) break;
                    const uint32_t bar = ragged ? land : full(v, n);
                    if (issue) {
                        mbar_expect_tx(bar, BYTES);
                        load_tile<DP>(slot(v, n), v ? maps.v : maps.k, bar, k0, hk, b);
                    }
                    const uint32_t bit = 1u << (v ? L::KS + n % L::VS : n % L::KS);
                    flying = ragged ? flying & ~bit : flying | bit;
                    parity = turn(v, n) ? parity | bit : parity & ~bit;
                    if (!ragged) continue;
                    ok = warp_wait(land, land_phase, abort_flag, limit);
                    land_open = !ok;
                    if (!ok) break;
                    land_phase ^= 1u;
                    clear_rows<DP>(slot(v, n), k0, keys.sink, keys.lo, keys.hi);
                    if (issue) mbar_arrive(full(v, n));
                }
            }
            const long long start = clock64();
            while (!mbar_test(q_full, 0) && clock64() - start < WAIT_CYCLES) {
            }
            while (land_open && !mbar_test(land, land_phase) && clock64() - start < WAIT_CYCLES) {
            }
            for (int i = 0; i < L::KS + L::VS; ++i)
                while ((flying >> i & 1u) && !mbar_test(bars + 8u * i, parity >> i & 1u) && clock64() - start < WAIT_CYCLES) {
                }
        } else if (warp == 1 && steps > 0) {
            const bool issue = elect_one();
            bool ok = warp_wait(q_full, 0, abort_flag, limit);
            const uint64_t qd = score_desc(q_tile), gd = score_desc(g_tile);
            auto begin_s = [&](int n) {
                if (!warp_wait(full(0, n), turn(0, n), abort_flag, limit)) return false;
                tc_fence_after();
                mma_scores<DP, TILE>(issue, tmem + (n & 1) * TILE, qd, score_desc(slot(0, n)));
                if (issue) mma_commit(s_full(n));
                return true;
            };
            auto begin_dp = [&](int n) {
                if (!warp_wait(full(1, n), turn(1, n), abort_flag, limit)) return false;
                tc_fence_after();
                mma_scores<DP, TILE>(issue, tmem + 2 * TILE, gd, score_desc(slot(1, n)));
                if (issue) {
                    mma_commit(dp_full);
                    mma_commit(empty(1, n));
                }
                return true;
            };
            ok = ok && begin_s(0) && begin_dp(0) && (steps == 1 || begin_s(1));
            for (int n = 0; n < steps && ok; ++n) {
                // both warpgroups have moved their columns of dQ
                if (LONG && n > 0 && fresh(n)) ok = warp_wait(ds_ready(1), n & 1, abort_flag, limit);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    ok = ok && warp_wait(ds_ready(w), n & 1, abort_flag, limit);
                    if (!ok) break;
                    tc_fence_after();
                    mma_sums<DP, 64>(issue, tmem + 3 * TILE, tmem + 2 * TILE + 64 * w, desc_on(sum_desc<DP>(slot(0, n)), w * 64 * 128), !fresh(n) || w > 0);
                }
                if (!ok) break;
                if (issue) mma_commit(empty(0, n));
                if (n + 1 < steps) ok = begin_dp(n + 1);
                if (ok && n + 2 < steps) ok = begin_s(n + 2);
            }
            if (ok && issue) mma_commit(sums_full);
            if (issue) mma_commit(drain);
            const long long start = clock64();
            while (!mbar_test(drain, 0) && clock64() - start < WAIT_CYCLES) {
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(MANY));
        const int w = (warp - 4) >> 2, quarter = warp & 3, lane_row = quarter * 32 + lane, q = q0 + lane_row;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        const uint32_t dp_at = lanes + 2 * TILE + 64 * w;
        const float c = p.scale * kLog2e, gain = gain_of(st, bh, 1, b * p.Hk + hk);
        const int64_t at = (static_cast<int64_t>(b) * p.Hq + h) * st.pitch + q;
        const float minus = st.minus[at] - SHIFT + log2f(gain);  // P is wanted times the power of two alone
        float delta = st.delta[at];
        const int pos = q + off, first_pos = q0 + off, last_pos = min(q0 + TILE, seq.nq) - 1 + off;
        const int row_hi = q < seq.nq ? pos : -1, row_lo = p.window && pos >= p.window ? pos - p.window + 1 : 0;
        // a warpgroup has half of the columns of dQ
        const int c0 = w * DP / 2, cols = min(p.D - c0, DP / 2);
        const uint32_t dq_at = lanes + 3 * TILE + c0;
        auto kept_row = [&] { return kept_at(kept + (static_cast<int64_t>(bh) * tiles + q0 / TILE) * TILE * p.D, lane_row, c0); };
        bool ok = true;
        for (int n = 0; n < steps && ok; ++n) {
            const int k0 = list.tile(n) * TILE;
            ok = warp_wait(s_full(n), n >> 1 & 1, abort_flag, limit);
            if (LONG && ok && n > 0 && fresh(n)) {  // dP comes after the sums of the step before
                ok = warp_wait(dp_full, n & 1, abort_flag, limit);
                if (!ok) break;
                tc_fence_after();
                if (cols > 0) keep_sums<DP / 2>(dq_at, kept_row(), cols, n == DRAIN, 1.0f);
            }
            if (!ok) break;
            tc_fence_after();
            uint32_t r[64];
            load64(lanes + (n & 1) * TILE + 64 * w, r);
            if (k0 + TILE - 1 > first_pos || q0 + TILE > seq.nq || (p.window && last_pos - k0 >= p.window && k0 + TILE > p.sinks)) {
                const int hi = row_hi - k0 + 1 - 64 * w, lo = row_lo - k0 - 64 * w, sink = min(p.sinks - k0 - 64 * w, hi);
                keep(r, (below(hi) & ~below(lo)) | below(sink), (below(hi - 32) & ~below(lo - 32)) | below(sink - 32));
            }
            weights(r, c, [&](int) { return both(minus); });
            if (sees_one(p, pos)) {
#pragma unroll
                for (uint32_t& x : r) x = 0;
            }
            ok = warp_wait(dp_full, n & 1, abort_flag, limit);
            if (!ok) break;
            tc_fence_after();
            uint32_t d[64];
            load64(dp_at, d);
            if (steps == 1) {
                P2 sum = pack(0.0f, 0.0f);
#pragma unroll
                for (int e = 0; e < 64; e += 2)
                    sum = fma2(pack(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), pack(__uint_as_float(d[e]), __uint_as_float(d[e + 1])), sum);
                part[w * TILE + lane_row] = sum2(sum);
                __syncwarp();
                if (lane == 0) mbar_arrive(part_full);
                ok = warp_wait(part_full, 0, abort_flag, limit);
                if (!ok) break;
                delta = (part[lane_row] + part[TILE + lane_row]) / gain;
                if (w == 0) st.delta[at] = q < seq.nq ? delta : 0.0f;
            }
#pragma unroll
            for (int h2 = 0; h2 < 2; ++h2) {
                uint32_t f[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int i = 32 * h2 + 2 * e;
                    const P2 x = sub2(pack(__uint_as_float(d[i]), __uint_as_float(d[i + 1])), both(delta));
                    const float2 y = unpack(mul2(pack(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), x));
                    f[e] = half2_of(y.x, y.y);
                }
                tmem_st16(dp_at + 16 * h2, f);
            }
            arrive(ds_ready(w));
        }
        if (ok && steps > 0) ok = warp_wait(sums_full, 0, abort_flag, limit);
        tc_fence_after();
        if (ok && p.dq.p) {
            __half* row = q < p.Sq ? reinterpret_cast<__half*>(p.dq.p) + b * p.dq.b + q * p.dq.s + h * p.dq.h : nullptr;
            if (steps > 0) {
                const bool live = q < seq.nq;
                if (cols > 0)
                    store_row<DP / 2>(dq_at, p.scale / gain, live && row ? row + c0 : nullptr, cols, LONG && steps > DRAIN ? kept_row() : nullptr);
                if (row && !live && cols > 0) zero_row(row + c0, cols);
            } else if (row && cols > 0) {
                zero_row(row + c0, cols);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag && threadIdx.x == 0) atomicExch(status, QSML_E_TIMEOUT);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <typename K, typename... A>
qsml_status_t launch(Context* ctx, K kernel, const char* name, size_t smem, int64_t ctas, const A&... args) {
    if (ctas > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "qsml_attention_backward: dimensions too large");
    QSML_TRY_STATUS(check_cuda(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)), name));
    const cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), smem, ctx->stream, args...);
    if (e != cudaSuccess) return check_cuda(ctx, e, name);
    return after_launch(ctx, name);
}

template <int DP> qsml_status_t backward(Context* ctx, const Problem& p, const Stats& st) {
    BwdMaps maps;
    if (!make_head_map(&maps.q, p.q, p.D, p.Sq, p.Hq, p.B) || !make_head_map(&maps.k, p.k, p.D, p.Sk, p.Hk, p.B) ||
        !make_head_map(&maps.v, p.v, p.D, p.Sk, p.Hk, p.B) || !make_head_map(&maps.g, p.dout, p.D, p.Sq, p.Hq, p.B))
        return set_error(ctx, QSML_E_CUDA, "qsml_attention_backward: cuTensorMapEncodeTiled failed");
    // first, as it takes the deltas of rows with few keys
    const int tq = (p.Sq + TILE - 1) / TILE, tk = (p.Sk + TILE - 1) / TILE;
    Workspace ws(ctx);
    if (p.dq.p || p.dk.p) {
        float* kept = nullptr;
        if (p.dq.p) QSML_TRY_STATUS(get_kept(&ws, p, &kept));
        QSML_TRY_STATUS(launch(ctx, kept ? k_attention_dq<DP, true> : k_attention_dq<DP, false>, "k_attention_dq", Dq<DP>::SMEM, static_cast<int64_t>(tq) * p.Hq * p.B, p, maps, st, tq, kept, ctx->status));
    }
    if (!p.dk.p && !p.dv.p) return QSML_OK;
    // Parts of about as many steps each, so that the CTAs are three waves: with a tile a CTA the one with
    // the sinks took as long as all else (2 x 4096 tokens of 16 heads over 2, window 2048: 540 us).
    KeyParts kp{nullptr, nullptr, 1, 1, p.window ? std::min((p.sinks + TILE - 1) / TILE, tk) : 0, tk};
    const int64_t bh = static_cast<int64_t>(p.B) * p.Hk, most = static_cast<int64_t>(p.G) * tq;
    const int64_t usual = p.window ? std::min(most, static_cast<int64_t>(p.G) * (p.window / TILE + 2)) : most;
    const int64_t total = bh * (kp.sink_tiles * most + (tk - kp.sink_tiles) * usual);
    const int64_t chunk = std::max<int64_t>(8, total / (3 * static_cast<int64_t>(ctx->num_sms)));
    auto parts = [&](int64_t steps) { return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(64, steps / chunk))); };
    kp.many = parts(most);
    kp.few = parts(usual);
    const bool split = kp.few > 1 || (kp.sink_tiles && kp.many > 1);
    // the steps that a part may have
    auto longest = [&](int64_t steps, int n) { return (steps + n - 1) / n; };
    const int64_t reach = p.window ? std::min<int64_t>(most, static_cast<int64_t>(p.G) * (p.window / TILE + 3)) : most;
    const bool drained = longest(reach, kp.few) > DRAIN || (kp.sink_tiles && longest(most, kp.many) > DRAIN);
    for (float** to : {split ? &kp.sum : nullptr, drained ? &kp.kept : nullptr}) {
        void* m = nullptr;
        if (!to) continue;
        QSML_TRY_STATUS(ws.get(sizeof(float) * kp.slots() * bh * 2 * TILE * p.D, &m));
        *to = static_cast<float*>(m);
    }
    QSML_TRY_STATUS(launch(ctx, drained ? k_attention_dkv<DP, true> : k_attention_dkv<DP, false>, "k_attention_dkv", Dkv<DP>::SMEM, kp.slots() * bh, p, maps, st, kp, ctx->status));
    if (!split) return QSML_OK;
    if (4 * tk * bh > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "qsml_attention_backward: dimensions too large");
    const int tiles = kp.few > 1 ? tk : kp.sink_tiles;
    const cudaError_t e = launch_pdl(k_attention_dkv_join, dim3(static_cast<unsigned>(4 * tiles * bh), 2), dim3(256), 0, ctx->stream, p, kp, tiles);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_attention_dkv_join");
    return after_launch(ctx, "k_attention_dkv_join");
}

}  // namespace

bool tc_takes_backward(const Problem& p) {
    auto out = [](const View& v) { return !v.p || heads::rows_on(v, 2, 16); };
    return p.Sq > 0 && tc_takes(p) && mappable(p.dout, p.D, p.Sq, p.Hq, p.B) && out(p.dq) && out(p.dk) && out(p.dv);
}

qsml_status_t backward_tc(Context* ctx, const Problem& p) {
    Workspace ws(ctx);
    Stats st;
    st.pitch = (p.Sq + TILE - 1) / TILE * static_cast<int64_t>(TILE);
    const int64_t rows = static_cast<int64_t>(p.B) * p.Hq * st.pitch;
    const int64_t norms = static_cast<int64_t>(p.B) * (2 * static_cast<int64_t>(p.Hq) + p.Hk);
    void* m = nullptr;
    QSML_TRY_STATUS(ws.get(sizeof(float) * (2 * rows + norms), &m));
    st.minus = static_cast<float*>(m);  // rows is a multiple of 128
    st.delta = st.minus + rows;
    st.of_q = reinterpret_cast<unsigned*>(st.delta + rows);
    st.of_v = st.of_q + 2 * static_cast<int64_t>(p.B) * p.Hq;
    QSML_TRY_STATUS(check_cuda(ctx, cudaMemsetAsync(st.of_q, 0, norms * sizeof(unsigned), ctx->stream), "qsml_attention_backward"));
    const int64_t qblocks = rows / TILE, vblocks = static_cast<int64_t>(p.B) * p.Hk * ((p.Sk + TILE - 1) / TILE);
    if (qblocks + vblocks > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "qsml_attention_backward: dimensions too large");
    const cudaError_t e = launch_pdl(k_attention_prepare, dim3(static_cast<unsigned>(qblocks + vblocks)), dim3(256), 0, ctx->stream, p, st,
                                     static_cast<int>(qblocks));
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_attention_prepare");
    QSML_TRY_STATUS(after_launch(ctx, "k_attention_prepare"));
    return p.D <= 64 ? backward<64>(ctx, p, st) : backward<128>(ctx, p, st);
}

}  // namespace attn
}  // namespace qsml
