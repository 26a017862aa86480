// Attention on the tensor cores (binary16, heads of up to 128 columns).
//
// A CTA takes 128 queries of a head and goes once over the keys that they see, in tiles of 128.
// S = Q K^T goes to TMEM; 128 threads, a row each, turn it into P = 2^(S c - m c + 6) with the row's
// running maximum m and leave P as binary16 where S was; O += P V stays in TMEM.  P is multiplied
// in two parts, the first while the second's exponentials are computed.  A row's O and sum are
// multiplied by 2^((m_old - m) c) only where m has grown by more than 2^8 since they were last: P
// then stays below 2^14, and the factor 2^6 keeps weights down to 2^-20 of the largest in
// binary16's normal range; both cancel in the end.
// Bound by the way from S over P and P V to the next S (2400 cycles, of which the exponentials
// take 1024 and the products of 128 columns as many), which two CTAs on a SM walk in turn: each
// has half of TMEM and of shared memory, with 128 columns one tile of K and one of V, the next
// loaded while the other is in use.  Measured at 8192 tokens of 32 heads over 8, 128 columns, every
// earlier key visible: 492 us, 1120 TFLOP/s.  One CTA with two tiles of queries that share the loads: 495, but 67 us
// instead of 53 for one head of 4096 tokens; two buffers of S with 64 keys each: 609; a quarter
// of the exponentials on the FMA pipe: no gain.
// Warp 0 loads by TMA into a ring, warp 1 issues the MMAs, the second warpgroup has the rows and
// the registers that the first gives up.  Values that no row of the CTA sees are cleared in shared
// memory, since a weight of 0 does not cancel what is not finite.
#include "attention_tc.cuh"

namespace qsml {
namespace attn {
namespace {

constexpr int kThreads = 256;

template <int DP> struct Fwd {
    static constexpr int STAGES = DP == 128 ? 2 : 5;
    static constexpr int PARTS = 2;
    static constexpr int BARS = 2 * STAGES + 5 + PARTS;
    static constexpr uint32_t TMEM = 256;  // 128 columns of S, then DP of O
    static constexpr int FEW = 40, MANY = 216;  // registers a thread of the warpgroups, of 2 x 128
    static constexpr size_t SMEM = (1 + STAGES) * size_t(TileOf<DP>::BYTES) + 1024 + 8 * BARS + 16;
    static_assert(2 * (SMEM + 1024) <= 233472, "shared memory of two CTAs");
};

struct FwdMaps {
    HeadMap q, k, v;
};

template <int DP, bool LONG>
__global__ void __launch_bounds__(kThreads, 2)
    k_attention_tc(const __grid_constant__ Problem p, const __grid_constant__ FwdMaps maps, int tiles, float* kept, int* status) {
    using L = Fwd<DP>;
    constexpr int BYTES = TileOf<DP>::BYTES, STAGES = L::STAGES, PARTS = L::PARTS;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    const uint32_t q_tile = base;
    auto ring = [&](int s) { return base + (1 + s) * BYTES; };
    const uint32_t bars = base + (1 + STAGES) * BYTES;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (STAGES + s); };
    const uint32_t q_full = bars + 8u * (2 * STAGES), land = q_full + 8, drain = q_full + 16, o_full = q_full + 24, s_full = q_full + 32;
    auto p_full = [&](int part) { return q_full + 40 + 8u * part; };
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
        mbar_init(s_full, 1);
        for (int i = 0; i < PARTS; ++i) mbar_init(p_full(i), 4);  // one arrival a warp
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(L::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
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
    auto fresh = [](int n) { return LONG ? n % DRAIN == 0 : n == 0; };  // whether O begins with step n

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::FEW));
        if (warp == 0 && steps > 0) {
            const bool issue = elect_one();
            uint32_t land_phase = 0;
            bool ok = true, land_open = false;
            if (issue) {
                mbar_expect_tx(q_full, BYTES);
                load_tile<DP>(q_tile, maps.q, q_full, q0, h, b);
            }
            int stage = 0;
            uint32_t phase = 0, flying = 0;  // slots whose last load has no other wait
            for (int n = 0; n < steps && ok; ++n) {
                const int k0 = list.tile(n) * TILE;
                // rows of V that nobody sees
                const bool ragged = k0 + TILE > keys.hi || (k0 < keys.lo && k0 + TILE > keys.sink);
                for (int i = 0; i < 2; ++i) {
                    ok = warp_wait(empty(stage), phase ^ 1u, abort_flag, limit);
                    if (!ok) break;
                    if (i == 1 && ragged) {
                        if (issue) {
                            mbar_expect_tx(land, BYTES);
                            load_tile<DP>(ring(stage), maps.v, land, k0, hk, b);
                        }
                        ok = warp_wait(land, land_phase, abort_flag, limit);
                        land_open = !ok;
                        if (!ok) break;
                        land_phase ^= 1u;
                        clear_rows<DP>(ring(stage), k0, keys.sink, keys.lo, keys.hi);
                        if (issue) mbar_arrive(full(stage));
                        flying &= ~(1u << stage);
                    } else {
                        if (issue) {
                            mbar_expect_tx(full(stage), BYTES);
                            load_tile<DP>(ring(stage), i ? maps.v : maps.k, full(stage), k0, hk, b);
                        }
                        flying |= 1u << stage;
                    }
                    if (++stage == STAGES) stage = 0, phase ^= 1u;
                }
            }
            // every copy has landed before the CTA can exit: slots below `stage` were last loaded
            // in this phase, the others in the one before
            const long long t0 = clock64();
            while (!mbar_test(q_full, 0) && clock64() - t0 < WAIT_CYCLES) {
            }
            for (int s = 0; s < STAGES; ++s)
                while ((flying >> s & 1u) && !mbar_test(full(s), s < stage ? phase : phase ^ 1u) && clock64() - t0 < WAIT_CYCLES) {
                }
            while (land_open && !mbar_test(land, land_phase) && clock64() - t0 < WAIT_CYCLES) {
            }
        } else if (warp == 1 && steps > 0) {
            const bool issue = elect_one();
            bool ok = warp_wait(q_full, 0, abort_flag, limit);
            auto slot = [&](int i) { return i % STAGES; };
            auto turn = [&](int i) { return static_cast<uint32_t>(i / STAGES) & 1u; };
            // S = Q K^T of step n, after O += P V of the one before: MMAs are executed in the order of
            // their issue, so P has been read when S is written over it.
            for (int n = 0; n <= steps && ok; ++n) {
                if (n > 0) {
                    const int v = 2 * n - 1;
                    ok = warp_wait(full(slot(v)), turn(v), abort_flag, limit);
                    const uint64_t x = sum_desc<DP>(ring(slot(v)));
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) {
                        constexpr int N = TILE / PARTS;
                        ok = ok && warp_wait(p_full(part), (n - 1) & 1, abort_flag, limit);
                        if (!ok) break;
                        tc_fence_after();
                        mma_sums<DP, N>(issue, tmem + TILE, tmem + part * N / 2, desc_on(x, part * N * 128), !fresh(n - 1) || part > 0);
                    }
                    if (!ok) break;
                    if (issue) mma_commit(empty(slot(v)));
                }
                if (n == steps) break;
                ok = warp_wait(full(slot(2 * n)), turn(2 * n), abort_flag, limit);
                if (!ok) break;
                tc_fence_after();
                mma_scores<DP, TILE>(issue, tmem, score_desc(q_tile), score_desc(ring(slot(2 * n))));
                if (issue) {
                    mma_commit(s_full);
                    mma_commit(empty(slot(2 * n)));
                }
            }
            if (ok && issue) mma_commit(o_full);
            if (issue) mma_commit(drain);
            const long long t0 = clock64();
            while (!mbar_test(drain, 0) && clock64() - t0 < WAIT_CYCLES) {
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::MANY));
        const int quarter = warp & 3, q = q0 + quarter * 32 + lane;
        const uint32_t s_at = tmem + (static_cast<uint32_t>(quarter * 32) << 16), o_at = s_at + TILE;
        const float c = p.scale * kLog2e;
        // the row's keys: [row_lo, row_hi] and those below p.sinks
        const int pos = q + off;
        const int row_hi = q < seq.nq ? pos : -1, row_lo = p.window && pos >= p.window ? pos - p.window + 1 : 0;
        const int first_pos = q0 + off, last_pos = min(q0 + TILE, seq.nq) - 1 + off;
        float m = -INFINITY, l = 0.0f, m_kept = -INFINITY;  // m_kept: the maximum that the kept row goes by
        auto kept_row = [&] { return kept_at(kept + (static_cast<int64_t>(bh) * tiles + q0 / TILE) * TILE * p.D, q - q0, 0); };
        auto kept_factor = [&] { return m_kept == m ? 1.0f : exp2_fast((m_kept - m) * c); };
        bool ok = true;
        for (int n = 0; n < steps && ok; ++n) {
            const int k0 = list.tile(n) * TILE;
            ok = warp_wait(s_full, n & 1, abort_flag, limit);
            if (!ok) break;
            tc_fence_after();
            if (LONG && n > 0 && fresh(n)) {  // P V of the steps before had been added when S came
                keep_sums<DP>(o_at, kept_row(), p.D, n == DRAIN, kept_factor());
                m_kept = m;
            }
            uint32_t r[TILE];
#pragma unroll
            for (int g = 0; g < TILE; g += 32) tmem_ld32_start(s_at + g, r + g);
#pragma unroll
            for (int g = 0; g < TILE; g += 32) tmem_wait(r + g);
            const bool partial = k0 + TILE - 1 > first_pos || q0 + TILE > seq.nq ||
                                 (p.window && last_pos - k0 >= p.window && k0 + TILE > p.sinks);
            if (partial) {  // as bits: compares of every element became branches, 5 us a tile
                const int hi = row_hi - k0 + 1, lo = row_lo - k0, sink = min(p.sinks - k0, hi);
#pragma unroll
                for (int g = 0; g < TILE / 32; ++g) {
                    const uint32_t seen = (below(hi - 32 * g) & ~below(lo - 32 * g)) | below(sink - 32 * g);
#pragma unroll
                    for (int e = 0; e < 32; ++e) r[32 * g + e] = seen & (1u << e) ? r[32 * g + e] : 0xff800000u;
                }
            }
            float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < TILE; e += 8)
#pragma unroll
                for (int j = 0; j < 4; ++j) most[j] = max3(most[j], __uint_as_float(r[e + j]), __uint_as_float(r[e + j + 4]));
            const float top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
            const bool grow = (top - m) * c > 8.0f;  // also from -inf
            if (__any_sync(0xffffffffu, grow)) {
                const float f = grow ? exp2_fast((m - top) * c) : 1.0f;
                if (grow) m = top;
                l *= f;
                if (!fresh(n)) {  // the P V before had been added when S came
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
            // in turn: the exponent of a pair, the exponentials of the pair AHEAD before, sum and rounding
            // of that AHEAD before it, so that none of a warp's instructions waits for the one before
            constexpr int AHEAD = 4, PAIRS = TILE / 2;
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < PAIRS + 2 * AHEAD; ++e) {
                if (e < PAIRS) {
                    const float2 x = unpack(fma2(pack(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), c2, ref2));
                    r[2 * e] = __float_as_uint(x.x);
                    r[2 * e + 1] = __float_as_uint(x.y);
                }
                if (e >= AHEAD && e < PAIRS + AHEAD) {
                    const int k = 2 * (e - AHEAD);
                    r[k] = __float_as_uint(exp2_fast(__uint_as_float(r[k])));
                    r[k + 1] = __float_as_uint(exp2_fast(__uint_as_float(r[k + 1])));
                }
                if (e >= 2 * AHEAD) {
                    const int k = e - 2 * AHEAD;
                    const float e0 = __uint_as_float(r[2 * k]), e1 = __uint_as_float(r[2 * k + 1]);
                    sum[k & 1] = add2(sum[k & 1], pack(e0, e1));
                    w[k % 16] = half2_of(e0, e1);
                    if (k % 16 == 15) tmem_st16(s_at + k - 15, w);
                    if ((k + 1) % (PAIRS / PARTS) == 0) {
                        tmem_st_wait();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_full((k + 1) / (PAIRS / PARTS) - 1));
                    }
                }
            }
            l += sum2(add2(sum[0], sum[1]));
        }
        const bool begun = steps > 0;
        if (ok && begun) ok = warp_wait(o_full, 0, abort_flag, limit);
        tc_fence_after();
        if (ok) {
            __half* to = q < p.Sq ? reinterpret_cast<__half*>(p.o.p) + b * p.o.b + q * p.o.s + h * p.o.h : nullptr;
            const bool any = l > 0.0f || isnan(l);
            if (begun)
                store_row<DP>(o_at, any ? 1.0f / l : 0.0f, to, p.D, LONG && steps > DRAIN ? kept_row() : nullptr, LONG ? kept_factor() : 1.0f);
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
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::TMEM) : "memory");
    }
}

template <int DP> qsml_status_t forward(Context* ctx, const Problem& p) {
    using L = Fwd<DP>;
    FwdMaps maps;
    if (!make_head_map(&maps.q, p.q, p.D, p.Sq, p.Hq, p.B) || !make_head_map(&maps.k, p.k, p.D, p.Sk, p.Hk, p.B) ||
        !make_head_map(&maps.v, p.v, p.D, p.Sk, p.Hk, p.B))
        return set_error(ctx, QSML_E_CUDA, "qsml_attention: cuTensorMapEncodeTiled failed");
    const char* name = "k_attention_tc";
    const int tiles = (p.Sq + TILE - 1) / TILE;
    if (static_cast<int64_t>(tiles) * p.Hq * p.B > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "qsml_attention: dimensions too large");
    Workspace ws(ctx);
    float* kept = nullptr;
    QSML_TRY_STATUS(get_kept(&ws, p, &kept));
    const auto kernel = kept ? k_attention_tc<DP, true> : k_attention_tc<DP, false>;
    QSML_TRY_STATUS(check_cuda(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(L::SMEM)), name));
    const cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(tiles * p.Hq * p.B)), dim3(kThreads), L::SMEM, ctx->stream, p, maps, tiles,
                                     kept, ctx->status);
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
