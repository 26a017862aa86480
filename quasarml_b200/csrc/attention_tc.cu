// Attention on the tensor cores (binary16, heads of up to 128 columns).
//
// A CTA takes 256 queries of a head as two tiles of 128 and goes once over the keys that they
// see, in units of 64.  For each unit and tile of queries S = Q K^T goes to TMEM; 128 threads, a
// row each, turn it into P = 2^(S c - m c + 6) with the row's running maximum m and leave P as
// binary16 where S was; O += P V stays in TMEM.  Each tile has two buffers of S, so the scores
// of the next unit are there before the exponentials of this one are done: with one buffer of
// 128 keys (all that TMEM holds beside two O of 128 columns) the way from S over P and P V to the
// next S was the bound.  A row's O and sum are multiplied by 2^((m_old - m) c) only where m has
// grown by more than 2^8 since they were last: P then stays below 2^14, and the factor 2^6 keeps
// weights down to 2^-20 of the largest in binary16's normal range; both cancel in the end.
// Bound by the exponentials (16 a cycle and SM, as many cycles as the two products of 128
// columns take) and by the tensor core.
// Warp 0 loads tiles of 128 keys by TMA into a ring, warp 1 issues the MMAs, warps 4-7 and 8-11
// have the rows of the two tiles and the registers that the first warpgroup gives up (64 + 2 x 208
// of 3 x 168).  Values that no row of the CTA sees are cleared in shared memory, since a weight of
// 0 does not cancel what is not finite.
#include "attention_tc.cuh"

namespace qsml {
namespace attn {
namespace {

constexpr int kThreads = 384;

template <int DP> struct Fwd {
    static constexpr int UNIT = DP == 128 ? 128 : 64;
    static constexpr int STAGES = DP == 128 ? 4 : 8;
    static constexpr int BARS = 2 * STAGES + 12;
    static constexpr size_t SMEM = (2 + STAGES) * size_t(TileOf<DP>::BYTES) + 1024 + 8 * BARS + 16;
    static_assert(SMEM <= 232448, "shared memory");
};

struct FwdMaps {
    HeadMap q, k, v;
};

// The keys of one tile of 128 queries that starts at q0, empty where no query is there.
__device__ __forceinline__ Keys keys_of(const Problem& p, const Seq& s, int q0) {
    const int off = s.nk - s.nq, last = min(q0 + TILE, s.nq) - 1;
    Keys k(p, s.nk, q0 + off, q0 < s.nq ? last + off : -1);
    if (q0 >= s.nq) k.sink = k.lo = k.hi = 0;
    return k;
}
// Whether any of the unit's keys is among them.
template <int UNIT> __device__ __forceinline__ bool meets(const Keys& k, int k0) { return k0 < k.hi && (k0 + UNIT > k.lo || k0 < k.sink); }

template <int DP>
__global__ void __launch_bounds__(kThreads, 1)
    k_attention_tc(const __grid_constant__ Problem p, const __grid_constant__ FwdMaps maps, int tiles, int* status) {
    using L = Fwd<DP>;
    constexpr int BYTES = TileOf<DP>::BYTES, STAGES = L::STAGES, UNIT = L::UNIT, PER = TILE / UNIT;  // units a tile of keys, and buffers of S
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    auto q_tile = [&](int t) { return base + t * BYTES; };
    auto ring = [&](int s) { return base + (2 + s) * BYTES; };
    const uint32_t bars = base + (2 + STAGES) * BYTES;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (STAGES + s); };
    const uint32_t q_full = bars + 8u * (2 * STAGES), land = q_full + 8, drain = q_full + 16, o_full = q_full + 24;
    auto s_full = [&](int t, uint32_t i) { return q_full + 32 + 16u * t + 8u * (i % PER); };  // the i-th unit of a tile
    auto p_full = [&](int t) { return q_full + 64 + 8u * t; };
    auto o_done = [&](int t) { return q_full + 80 + 8u * t; };
    unsigned char* misc = smem_raw + (bars - raw) + 8 * L::BARS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        mbar_init(q_full, 1);
        mbar_init(land, 1);
        mbar_init(drain, 1);
        mbar_init(o_full, 1);
        for (int t = 0; t < 2; ++t) {
            mbar_init(s_full(t, 0), 1);
            mbar_init(s_full(t, 1), 1);
            mbar_init(p_full(t), 4);  // one arrival a warp
            mbar_init(o_done(t), 1);
        }
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
    const uint32_t tmem = *tmem_slot;
    pdl_begin();
    const long long limit = wait_limit(status);

    // the last queries, with the most keys, first
    const int b = blockIdx.x / p.Hq / tiles, rest = blockIdx.x - b * p.Hq * tiles;
    const int q0 = (tiles - 1 - rest / p.Hq) * 2 * TILE, h = rest % p.Hq, hk = h / p.G;
    const Seq seq(p, b);
    const int off = seq.nk - seq.nq;
    const Keys keys[2] = {keys_of(p, seq, q0), keys_of(p, seq, q0 + TILE)};
    Keys both_tiles(p, seq.nk, q0 + off, min(q0 + 2 * TILE, seq.nq) - 1 + off);
    const Tiles list(both_tiles, TILE);
    const int steps = q0 < seq.nq ? list.n : 0;

    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 0) {
        int issued[STAGES];
#pragma unroll
        for (int s = 0; s < STAGES; ++s) issued[s] = -1;
        uint32_t land_phase = 0;
        bool ok = steps > 0, land_open = false;
        if (ok && lane == 0) {
            const int n = q0 + TILE < seq.nq ? 2 : 1;
            mbar_expect_tx(q_full, n * BYTES);
            for (int t = 0; t < n; ++t) load_tile<DP>(q_tile(t), maps.q, q_full, q0 + t * TILE, h, b);
        }
        int stage = 0;
        uint32_t phase = 0;
        for (int n = 0; n < steps && ok; ++n) {
            const int k0 = list.tile(n) * TILE;
            // rows of V that nobody sees
            const bool ragged = k0 + TILE > both_tiles.hi || (k0 < both_tiles.lo && k0 + TILE > both_tiles.sink);
            for (int i = 0; i < 2 && ok; ++i) {
                ok = warp_wait(empty(stage), phase ^ 1u, abort_flag, limit);
                if (!ok) break;
                if (i == 1 && ragged) {
                    if (lane == 0) {
                        mbar_expect_tx(land, BYTES);
                        load_tile<DP>(ring(stage), maps.v, land, k0, hk, b);
                    }
                    ok = warp_wait(land, land_phase, abort_flag, limit);
                    land_open = !ok;
                    if (!ok) break;
                    land_phase ^= 1u;
                    clear_rows<DP>(ring(stage), k0, both_tiles.sink, both_tiles.lo, both_tiles.hi);
                    if (lane == 0) mbar_arrive(full(stage));
                    issued[stage] = -1;  // landed already
                } else if (lane == 0) {
                    mbar_expect_tx(full(stage), BYTES);
                    load_tile<DP>(ring(stage), i ? maps.v : maps.k, full(stage), k0, hk, b);
                    issued[stage] = static_cast<int>(phase);
                }
                if (++stage == STAGES) stage = 0, phase ^= 1u;
            }
        }
        // every copy has landed before the CTA can exit
        if (lane == 0 && steps > 0) {
            const long long t0 = clock64();
            while (!mbar_test(q_full, 0) && clock64() - t0 < WAIT_CYCLES) {
            }
#pragma unroll
            for (int s = 0; s < STAGES; ++s)
                while (issued[s] >= 0 && !mbar_test(full(s), static_cast<uint32_t>(issued[s])) && clock64() - t0 < WAIT_CYCLES) {
                }
            while (land_open && !mbar_test(land, land_phase) && clock64() - t0 < WAIT_CYCLES) {
            }
        }
    } else if (warp == 1) {
        if (steps > 0) {
            const bool issue = elect_one();
            bool ok = warp_wait(q_full, 0, abort_flag, limit);
            int waiting[2] = {-1, -1};    // unit whose P is still to be multiplied
            uint32_t count[2] = {0, 0};   // units begun
            auto slot = [&](int i) { return i % STAGES; };
            auto turn = [&](int i) { return static_cast<uint32_t>(i / STAGES) & 1u; };
            // With two buffers of S the order is Q K of both tiles, then P V of their units before, with
            // one P V before Q K: P has been read when the next S is written to its buffer, MMAs being
            // executed in the order of their issue.
            auto sums = [&](int t) {
                const int v = 2 * (waiting[t] / PER) + 1, i = static_cast<int>(count[t]) - 1;
                if (!warp_wait(p_full(t), i & 1, abort_flag, limit) || !warp_wait(full(slot(v)), turn(v), abort_flag, limit)) return false;
                tc_fence_after();
                mma_sums<DP, UNIT>(issue, tmem + 256 + t * DP, tmem + t * TILE + i % PER * UNIT,
                                   desc_on(sum_desc<DP>(ring(slot(v))), waiting[t] % PER * UNIT * 128), i > 0);
                if (issue) mma_commit(o_done(t));
                return true;
            };
            for (int u = 0; u < PER * steps && ok; ++u) {
                const int n = u / PER, k0 = list.tile(n) * TILE + u % PER * UNIT;
                if (u % PER == 0) {
                    ok = warp_wait(full(slot(2 * n)), turn(2 * n), abort_flag, limit);
                    if (!ok) break;
                    tc_fence_after();
                }
                const bool now[2] = {meets<UNIT>(keys[0], k0), meets<UNIT>(keys[1], k0)};
                auto scores = [&](int t) {
                    if (!now[t]) return;
                    mma_scores<DP, UNIT>(issue, tmem + t * TILE + count[t] % PER * UNIT, score_desc(q_tile(t)),
                                         desc_on(score_desc(ring(slot(2 * n))), u % PER * UNIT * 128));
                    if (issue) mma_commit(s_full(t, count[t]));
                };
                if (PER > 1) scores(0), scores(1);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (ok && waiting[t] >= 0) ok = sums(t);
                    if (PER == 1 && ok) scores(t);
                    waiting[t] = now[t] ? u : -1;
                    count[t] += now[t];
                }
                if (ok && issue) {
                    if (u % PER == PER - 1) mma_commit(empty(slot(2 * n)));
                    if (u % PER == 0 && n > 0) mma_commit(empty(slot(2 * n - 1)));
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (ok && waiting[t] >= 0) ok = sums(t);
            if (ok && issue) mma_commit(o_full);
            if (issue) mma_commit(drain);
            const long long t0 = clock64();
            while (!mbar_test(drain, 0) && clock64() - t0 < WAIT_CYCLES) {
            }
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int t = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t o_at = tmem + lanes + 256 + t * DP;
        const int qt = q0 + t * TILE, q = qt + row;
        const float c = p.scale * kLog2e;
        // the row's keys: [row_lo, row_hi] and those below row_sink
        const int pos = q + off;
        const bool there = q < seq.nq;
        const int row_hi = there ? pos : -1, row_lo = p.window && pos >= p.window ? pos - p.window + 1 : 0;
        const int first_pos = qt + off, last_pos = min(qt + TILE, seq.nq) - 1 + off;
        float m = -INFINITY, l = 0.0f;
        uint32_t i = 0;  // units done
        bool ok = true;
        for (int u = 0; u < PER * steps && ok; ++u) {
            const int k0 = list.tile(u / PER) * TILE + u % PER * UNIT;
            if (!meets<UNIT>(keys[t], k0)) continue;
            ok = warp_wait(s_full(t, i), i / PER & 1u, abort_flag, limit);
            if (!ok) break;
            tc_fence_after();
            const uint32_t s_at = tmem + lanes + t * TILE + i % PER * UNIT;
            uint32_t r[UNIT];
#pragma unroll
            for (int g = 0; g < UNIT; g += 32) tmem_ld32_start(s_at + g, r + g);
#pragma unroll
            for (int g = 0; g < UNIT; g += 32) tmem_wait(r + g);
            const bool partial = k0 + UNIT - 1 > first_pos || qt + TILE > seq.nq ||
                                 (p.window && last_pos - k0 >= p.window && k0 + UNIT > p.sinks);
            if (partial) {
                const int hi = row_hi - k0 + 1, lo = row_lo - k0, sink = min(p.sinks - k0, hi);
#pragma unroll
                for (int g = 0; g < UNIT / 32; ++g) {
                    const uint32_t seen = (below(hi - 32 * g) & ~below(lo - 32 * g)) | below(sink - 32 * g);
#pragma unroll
                    for (int e = 0; e < 32; ++e) r[32 * g + e] = seen & (1u << e) ? r[32 * g + e] : 0xff800000u;
                }
            }
            float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < UNIT; e += 8)
#pragma unroll
                for (int j = 0; j < 4; ++j) most[j] = max3(most[j], __uint_as_float(r[e + j]), __uint_as_float(r[e + j + 4]));
            const float top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
            const bool grow = (top - m) * c > 8.0f;  // also from -inf
            if (__any_sync(0xffffffffu, grow)) {
                const float f = grow ? exp2_fast((m - top) * c) : 1.0f;
                if (grow) m = top;
                l *= f;
                if (i > 0) {
                    // the products before have been added (those of the unit before that had, when S came)
                    ok = warp_wait(o_done(t), (i - 1) & 1u, abort_flag, limit);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int d = 0; d < DP; d += 32) {
                        uint32_t o[32];
                        tmem_ld32(o_at + d, o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st32(o_at + d, o);
                    }
                }
            }
            const float ref = 6.0f - (m == -INFINITY ? 0.0f : m * c);
            const P2 c2 = both(c), ref2 = both(ref);
            P2 sum[2] = {pack(0.0f, 0.0f), pack(0.0f, 0.0f)};
#pragma unroll
            for (int g = 0; g < UNIT / 32; ++g) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int at = 32 * g + 2 * e;
                    const float2 x = unpack(fma2(pack(__uint_as_float(r[at]), __uint_as_float(r[at + 1])), c2, ref2));
                    const float e0 = exp2_fast(x.x), e1 = exp2_fast(x.y);
                    sum[e & 1] = add2(sum[e & 1], pack(e0, e1));
                    w[e] = half2_of(e0, e1);
                }
                tmem_st16(s_at + 16 * g, w);
            }
            l += sum2(add2(sum[0], sum[1]));
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(t));
            ++i;
        }
        const bool begun = i > 0;
        if (ok && begun) ok = warp_wait(o_full, 0, abort_flag, limit);
        tc_fence_after();
        if (ok && qt < p.Sq) {
            __half* to = q < p.Sq ? reinterpret_cast<__half*>(p.o.p) + b * p.o.b + q * p.o.s + h * p.o.h : nullptr;
            const bool any = l > 0.0f || isnan(l);
            if (begun)
                store_row<DP>(o_at, any ? 1.0f / l : 0.0f, to, p.D);
            else if (to)
                zero_row(to, p.D);
            if (p.lse && q < p.Sq)
                p.lse[(static_cast<int64_t>(b) * p.Hq + h) * p.Sq + q] = any ? (m * c - 6.0f + log2f(l)) * kLn2 : -INFINITY;
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

template <int DP> qsml_status_t forward(Context* ctx, const Problem& p) {
    FwdMaps maps;
    if (!make_head_map(&maps.q, p.q, p.D, p.Sq, p.Hq, p.B) || !make_head_map(&maps.k, p.k, p.D, p.Sk, p.Hk, p.B) ||
        !make_head_map(&maps.v, p.v, p.D, p.Sk, p.Hk, p.B))
        return set_error(ctx, QSML_E_CUDA, "qsml_attention: cuTensorMapEncodeTiled failed");
    const char* name = "k_attention_tc";
    const int tiles = (p.Sq + 2 * TILE - 1) / (2 * TILE);
    if (static_cast<int64_t>(tiles) * p.Hq * p.B > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "qsml_attention: dimensions too large");
    QSML_TRY_STATUS(check_cuda(ctx, cudaFuncSetAttribute(k_attention_tc<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Fwd<DP>::SMEM)), name));
    const cudaError_t e = launch_pdl(k_attention_tc<DP>, dim3(static_cast<unsigned>(tiles * p.Hq * p.B)), dim3(kThreads), Fwd<DP>::SMEM, ctx->stream,
                                     p, maps, tiles, ctx->status);
    if (e != cudaSuccess) return check_cuda(ctx, e, name);
    return after_launch(ctx, name);
}

}  // namespace

bool tc_takes(const Problem& p) {
    return p.f16 && p.Sk > 0 && mappable(p.q, p.D, p.Sq, p.Hq, p.B) && mappable(p.k, p.D, p.Sk, p.Hk, p.B) &&
           mappable(p.v, p.D, p.Sk, p.Hk, p.B) && heads::rows_on(p.o, 2, 16);
}

qsml_status_t forward_tc(Context* ctx, const Problem& p) { return p.D <= 64 ? forward<64>(ctx, p) : forward<128>(ctx, p); }

}  // namespace attn
}  // namespace qsml
