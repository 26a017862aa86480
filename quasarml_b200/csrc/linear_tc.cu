// The linear layers' products on the tensor cores (tcgen05.mma, accumulators in
// TMEM, operands staged by TMA in 128-byte swizzled shared memory).
//
// Operands are tiles of 128 rows (of the result's rows or columns) by 64 k in
// 16-bit elements, 16 KiB, in whichever order they lie in memory: K-major (k
// contiguous: one box of 64 k x 128) or MN-major (two boxes of 64 x 64 k).  So x
// and x^T, w and w^T are read in place by the forward product, dz w^T and x^T dz.
// Operands that TMA cannot read (a row pitch or start off 16 bytes, strides in
// both dims) are copied once to a workspace.
//
// binary16: one product, kind::f16, binary32 accumulators; an operand that comes in
// two parts (its value their sum) is two segments of the sum.  A tensor-core accumulator
// is truncated at each step, so one stands for no more than 8192 k: sums of one sign lose
// 5e-5 of theirs so (measured; with 16384 k 1.0e-4, with 131072 8.4e-4, more than
// binary16's rounding).  The accumulators of a longer sum are added, to the nearest, in a
// second one.
// binary32: x = x0 + x1 + x2 exactly, three bf16 parts of 8 bits each (the upper
// bits by truncation, so no part overflows and all have x's sign); the six
// products x_i w_j with i + j <= 2 are formed on the bf16 pipe.  x1 is below 2^-7 |x| and
// x2 below 2^-15 |x|, so the dropped ones are below 2^-21 |x w| together (7.83 * 2^-24 at
// x = w = 1 + 2^-7 - 2^-23); they have the product's sign, so that sums of one sign lose
// 0.7 * 2^-24 of theirs in the mean.  The accumulators are truncated here too: the main
// product x0 w0 is drained every 256 k into binary32 registers (rounded to nearest
// there); the other five, 2^-7 of it and less, have an accumulator of their own, drained
// every 2048 k: sums of one sign lose 3e-7 of theirs (measured at 131072 k, where one
// accumulator for the whole sum lost 1.9e-5).  Cost: six times binary16's.
//
// k_linear_tc: 128 x 128 of the result a CTA (64 columns of each weight for a dual
// product).  Where the tiles do not fill the GPU, a cluster of up to 8 CTAs splits
// the sum over k: each leaves its binary32 tile in shared memory, and all of them
// add the cluster's tiles, in rank order, for a share of the outputs (distributed
// shared memory: no workspace, no atomics, one launch).
#include "linear.cuh"
#include "tcgen05.cuh"

namespace qsml {
namespace linear {
namespace {

using namespace tc;

constexpr int TILE_BYTES = 128 * 128;     // one operand tile: 128 rows x 64 k
constexpr int CHUNK = 4;                  // binary32: k-blocks between drains
constexpr int LESSER = 8;                 // binary32: drains of the main product to one of the lesser ones
static_assert(LESSER >= 2, "two columns of lesser products in turn");
constexpr int LONG = 128;                 // binary16: k-blocks that one accumulator stands for
constexpr int THREADS = 192;              // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue
constexpr int MAX_SPLIT = 8;              // portable cluster size

struct TcArgs {
    CUtensorMap a[2], b[2];
    Epilogue e;
    int M, N;
    int tiles_m, tiles_n;
    int kb;                  // k-blocks of 64 a segment
    int segments;            // binary16 with an operand in two parts: twice the problem's
    int halves;              // then 2, else 1
    int a_halves, b_halves;  // which operand it is
    int splits;
    int a_bytes;             // k_linear_tc: of an operand tile of A (fewer than 128 rows where M has fewer)
    int slots, ring;         // k_linear_tc: operand tiles of A and B in the ring, and its bytes
    int a_mn[2], b_mn[2];    // MN-major operands, by segment
    int* status;
};
// The products of one launch: g[i]'s CTAs begin at CTA first[i].
template <int NP> struct TcBatch {
    TcArgs g[NP];
    int first[NP];
};

// A ring of slots in shared memory, each a tile of A and one of B (of one part, for
// binary32: a k-block takes three).  Binary16 has two CTAs a SM with 96 KiB each, or
// one with 192 KiB where there are no more CTAs than SMs (three slots do not cover
// L2's latency: 512 x 11008 x 4096 took 70 us, with six 45; 256 x 11008 x 4096 42 and
// 30).
template <bool F32> struct Shape {
    static constexpr int PARTS = F32 ? 3 : 1;
    static constexpr int MAX_SLOTS = 6;
    static constexpr int TMEM = F32 ? 256 : 128;  // columns; twice that for binary32 and long sums
    static constexpr int RING = F32 ? 6 * 32768 : 3 * 32768;
    static constexpr int DEEP_RING = 6 * 32768;
    static constexpr int BARS = 8 * (2 * MAX_SLOTS + 5) + 8;
    static constexpr size_t smem(int ring) { return size_t(ring) + 1024 + BARS; }
    static constexpr int CTAS = F32 ? 1 : 2;  // a SM
};

// D f32; A and B f16 (0) or bf16 (1); their major-ness; N, M.
__device__ __forceinline__ uint32_t idesc(bool bf16, int a_mn, int b_mn, int m, int n) {
    const uint32_t f = bf16 ? 1u : 0u;
    return (1u << 4) | (f << 7) | (f << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) | (uint32_t(n >> 3) << 17) |
           (uint32_t(m >> 4) << 24);
}

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
}

// total (or nothing, for the first) + the 32 columns at `from`, each in this thread's lane, to
// `total`: binary32 additions to the nearest.
__device__ __forceinline__ void tmem_add32(uint32_t total, uint32_t from, bool first) {
    uint32_t v[32];
    tmem_ld32(from, v);
    if (!first) {
        uint32_t t[32];
        tmem_ld32(total, t);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__fadd_rn(__uint_as_float(t[i]), __uint_as_float(v[i])));
    }
    tmem_st32(total, v);
}

// The k16 slice k of a tile: K-major rows of 128 bytes (32 bytes a slice), or
// MN-major chunks of 64 with 128 bytes a k (2048 bytes a slice, chunks 8 KiB apart).
__device__ __forceinline__ uint64_t slice_desc(uint32_t tile, int mn, int k) {
    return mn ? smem_desc(tile + k * 2048, 8192, 1024) : smem_desc(tile + k * 32, 16, 1024);
}

// ---- the binary16 epilogue of a row, 32 columns in registers -----------------------
// z += bias of columns col .. col + 31 (the warp's lanes have one row each and read
// the same 32 values)
__device__ __forceinline__ void add_bias32(const Epilogue& e, int which, int64_t col, float (&z)[32]) {
    if (!e.bias[which]) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t c = col + 8 * j;
        if (c >= e.N) break;
        const int n = e.N - c < 8 ? static_cast<int>(e.N - c) : 8;
        float b[8];
        if (e.bias_f32) ldg8(static_cast<const float*>(e.bias[which]) + c, n, e.vec == 1, b);
        else ldg8(static_cast<const __half*>(e.bias[which]) + c, n, e.vec == 1, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) z[8 * j + i] = __fadd_rn(z[8 * j + i], b[i]);
    }
}

// A warp's staging buffer: 32 rows of COLS binary16 in 16-byte units, swapped by
// row so that a column of units and a row of them both meet every bank.
template <int COLS> struct HalfRows {
    static constexpr int UNITS = COLS / 8;
    static constexpr int BYTES = 32 * COLS * 2;
    uint32_t base;
    __device__ uint32_t at(int row, int unit) const {
        return base + row * (COLS * 2) + ((unit ^ ((COLS == 64 ? row : row >> 1) & (UNITS - 1))) << 4);
    }
    // 32 columns of the lane's row, from column 32 * h of the buffer on
    __device__ void put(int lane, int h, const float (&z)[32]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __half2 v = __floats2half2_rn(z[8 * j + 2 * i], z[8 * j + 2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&v);
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at(lane, 4 * h + j)), "r"(w[0]), "r"(w[1]),
                         "r"(w[2]), "r"(w[3])
                         : "memory");
        }
    }
    __device__ void add(int lane, int h, float (&z)[32]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t w[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(at(lane, 4 * h + j))
                         : "memory");
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                z[8 * j + 2 * i] = __fadd_rn(z[8 * j + 2 * i], f.x);
                z[8 * j + 2 * i + 1] = __fadd_rn(z[8 * j + 2 * i + 1], f.y);
            }
        }
    }
    // The buffer's rows to or from a matrix of N columns, rows of `ld`, whose element
    // (0, 0) lies at p; `rows` of the 32 exist.  Neighbouring lanes take neighbouring
    // units of a row (vec 1), pairs (2) or elements (0).
    template <bool LOAD>
    __device__ void copy(__half* p, int64_t ld, int64_t col, int64_t N, int64_t row0, int rows, int vec) const {
        if (vec == 1) move<LOAD, 8>(p + row0 * ld + col, ld, N - col, rows);
        else if (vec == 2) move<LOAD, 2>(p + row0 * ld + col, ld, N - col, rows);
        else move<LOAD, 1>(p + row0 * ld + col, ld, N - col, rows);
    }

private:
    // E elements a lane; the first `left` columns exist, a multiple of E
    template <bool LOAD, int E> __device__ void move(__half* p, int64_t ld, int64_t left, int rows) const {
        constexpr int LANES = COLS / E;  // of a row
        constexpr int STEPS = LANES > 32 ? LANES / 32 : 1, ROWS = LANES > 32 ? 1 : 32 / LANES;
        const int lane = threadIdx.x & 31, c0 = lane % LANES * E;
#pragma unroll 4
        for (int r = LANES > 32 ? 0 : lane / LANES; r < rows; r += ROWS)
#pragma unroll
            for (int j = 0; j < STEPS; ++j) {
                const int c = c0 + j * 32 * E;
                if (c >= left) continue;
                __half* q = p + r * ld + c;
                const uint32_t s = at(r, c / 8) + c % 8 * 2;
                if constexpr (E == 8) {
                    uint4 u;
                    if (LOAD) {
                        u = *reinterpret_cast<const uint4*>(q);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(s), "r"(u.x), "r"(u.y), "r"(u.z),
                                     "r"(u.w)
                                     : "memory");
                    } else {
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                                     : "r"(s)
                                     : "memory");
                        *reinterpret_cast<uint4*>(q) = u;
                    }
                } else if constexpr (E == 2) {
                    uint32_t u;
                    if (LOAD) {
                        u = *reinterpret_cast<const uint32_t*>(q);
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(s), "r"(u) : "memory");
                    } else {
                        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(u) : "r"(s) : "memory");
                        *reinterpret_cast<uint32_t*>(q) = u;
                    }
                } else {
                    uint16_t u;
                    if (LOAD) {
                        u = *reinterpret_cast<const uint16_t*>(q);
                        asm volatile("st.shared.b16 [%0], %1;" ::"r"(s), "h"(u) : "memory");
                    } else {
                        asm volatile("ld.shared.b16 %0, [%1];" : "=h"(u) : "r"(s) : "memory");
                        *reinterpret_cast<uint16_t*>(q) = u;
                    }
                }
            }
    }
};

// From a k slice's descriptor to the next.
__device__ __forceinline__ constexpr uint32_t slice_step(int mn) { return mn ? 2048u >> 4 : 32u >> 4; }

// f(a_mn, b_mn) with the orders as constants: the MMA thread issues an MMA every 64
// to 128 cycles alone, and descriptors whose steps it has to look up cost 10 % of a
// large product (227 us against 205 at 8192 x 4096 x 4096).
template <class F> __device__ __forceinline__ void by_order(int a_mn, int b_mn, F&& f) {
    using No = std::integral_constant<int, 0>;
    using Yes = std::integral_constant<int, 1>;
    if (a_mn) {
        if (b_mn) f(Yes{}, Yes{});
        else f(Yes{}, No{});
    } else {
        if (b_mn) f(No{}, Yes{});
        else f(No{}, No{});
    }
}

// The producer and MMA warps run their loops with all lanes, so that addresses and
// descriptors stay in uniform registers; one lane of them issues.
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, long long limit) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, limit)) != 0;
}

__device__ __forceinline__ void cluster_arrive_wait() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

__device__ __forceinline__ int ld_cluster1(uint32_t addr) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ float lds1(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 lds4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

template <bool F32, bool DUAL, int NP>
__global__ void __launch_bounds__(THREADS, Shape<F32>::CTAS) k_linear_tc(const __grid_constant__ TcBatch<NP> all) {
    int which = 0;
    for (int i = 1; i < NP; ++i)
        if (static_cast<int>(blockIdx.x) >= all.first[i]) which = i;
    const int cta = static_cast<int>(blockIdx.x) - (NP > 1 ? all.first[which] : 0);
    const TcArgs& g = all.g[which];
    using T = std::conditional_t<F32, float, __half>;
    using S = Shape<F32>;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char* gbase = smem_raw + (base - raw);
    const uint32_t bars = base + g.ring;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (S::MAX_SLOTS + s); };
    auto tfull_bar = [&](int a) { return bars + 8u * (2 * S::MAX_SLOTS + a); };
    auto tempty_bar = [&](int a) { return bars + 8u * (2 * S::MAX_SLOTS + 2 + a); };
    const uint32_t drain_bar = bars + 8u * (2 * S::MAX_SLOTS + 4);
    unsigned char* misc = gbase + g.ring + 8 * (2 * S::MAX_SLOTS + 5);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 4);

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int tile = cta / g.splits, rank = cta % g.splits;
    const int mt = tile % g.tiles_m, nt = tile / g.tiles_m;
    constexpr int BN = DUAL ? 64 : 128;  // result columns a tile
    // this CTA's share of the k-blocks, and of it the part [lo, hi) in segment seg
    const int total = g.kb * g.segments;
    const int u0 = static_cast<int>(static_cast<int64_t>(total) * rank / g.splits);
    const int u1 = static_cast<int>(static_cast<int64_t>(total) * (rank + 1) / g.splits);
    auto part = [&](int seg, int& lo, int& hi) {
        lo = min(max(u0 - seg * g.kb, 0), g.kb);
        hi = min(max(u1 - seg * g.kb, 0), g.kb);
    };
    // binary16: the accumulators of the CTA's sum, added up behind the first 128 columns
    const int sums = (u1 - u0 + LONG - 1) / LONG;
    const uint32_t tmem_cols = F32 || sums > 1 ? 2 * S::TMEM : S::TMEM;
    if (threadIdx.x == 0) {
        for (int s = 0; s < g.slots; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), 4);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_begin();  // everything above needed no memory of the kernels before
    const long long limit = wait_limit(g.status);

    // A's tile comes first: where it has fewer than 128 rows the MMA takes the rest
    // from B's, for rows of the result that are not there
    const uint32_t slot_bytes = g.a_bytes + TILE_BYTES;

    bool done = true;  // epilogue warps: the CTA's sums are complete
    if (warp == 0) {
        const bool issue = elect_one();
        int slot = 0, filled = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int sp = 0; sp < g.segments && ok; ++sp) {
            const int seg = sp / g.halves, half = sp - seg * g.halves;
            int lo, hi;
            part(sp, lo, hi);
            by_order(g.a_mn[seg], g.b_mn[DUAL ? 0 : seg], [&](auto a_mn, auto b_mn) {
                const int ha = g.a_halves ? half : 0, hb = g.b_halves ? half : 0;
                const CUtensorMap* ma = &g.a[seg];
                [[maybe_unused]] const CUtensorMap* mb = &g.b[DUAL ? 0 : seg];
                for (int kb = lo; kb < hi && ok; ++kb) {
#pragma unroll
                    for (int p = 0; p < S::PARTS; ++p) {
                        if (!warp_wait(empty_bar(slot), phase ^ 1u, abort_flag, limit)) {
                            ok = false;
                            break;
                        }
                        const uint32_t bar = full_bar(slot), at = base + slot * slot_bytes, bt = at + g.a_bytes;
                        if (issue) {
                            mbar_expect_tx(bar, slot_bytes);
                            if (a_mn.value) {
                                tma_load_3d(at, ma, bar, mt * 128, kb * 64, F32 ? p : ha);
                                tma_load_3d(at + 8192, ma, bar, mt * 128 + 64, kb * 64, F32 ? p : ha);
                            } else {
                                tma_load_3d(at, ma, bar, kb * 64, mt * 128, F32 ? p : ha);
                            }
                            if constexpr (DUAL) {
#pragma unroll
                                for (int j = 0; j < 2; ++j) {
                                    if (b_mn.value) tma_load_3d(bt + j * 8192, &g.b[j], bar, nt * 64, kb * 64, F32 ? p : hb);
                                    else tma_load_3d(bt + j * 8192, &g.b[j], bar, kb * 64, nt * 64, F32 ? p : hb);
                                }
                            } else if (b_mn.value) {
                                tma_load_3d(bt, mb, bar, nt * 128, kb * 64, F32 ? p : hb);
                                tma_load_3d(bt + 8192, mb, bar, nt * 128 + 64, kb * 64, F32 ? p : hb);
                            } else {
                                tma_load_3d(bt, mb, bar, kb * 64, nt * 128, F32 ? p : hb);
                            }
                        }
                        ++filled;
                        if (++slot == g.slots) {
                            slot = 0;
                            phase ^= 1u;
                        }
                    }
                }
            });
        }
        // every copy this thread started lands before the memory has another use:
        // the last fill of each slot (fill i is in slot i % slots, phase i / slots)
        for (int i = max(0, filled - g.slots); i < filled; ++i) {
            const uint32_t parity = static_cast<uint32_t>((i / g.slots) & 1);
            const long long t0 = clock64();
            while (!mbar_test(full_bar(i % g.slots), parity) && clock64() - t0 < WAIT_CYCLES) {
            }
        }
    } else if (warp == 1) {
        const bool issue = elect_one();
        int slot = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        uint32_t small = tmem + 256;  // binary32: the five lesser products, here or 128 columns on
        int drains = 0;               // of the main product, since the lesser ones' last
        bool begun = false;
        int blocks = 0;  // binary16: in the accumulator
        for (int sp = 0; sp < g.segments && ok; ++sp) {
            const int seg = sp / g.halves;
            int lo, hi;
            part(sp, lo, hi);
            by_order(g.a_mn[seg], g.b_mn[DUAL ? 0 : seg], [&](auto a_mn, auto b_mn) {
                const uint32_t id = idesc(F32, a_mn.value, b_mn.value, 128, 128);
                const uint64_t wa = slice_desc(base, a_mn.value, 0), wb = slice_desc(base + g.a_bytes, b_mn.value, 0);
                // binary32: a drain every CHUNK k-blocks; else none inside
                for (int k0 = lo; k0 < hi && ok; k0 += F32 ? CHUNK : hi) {
                    const int k1 = F32 ? min(k0 + CHUNK, hi) : hi;
                    if (F32) {
                        if (!warp_wait(tempty_bar(acc), acc_phase ^ 1u, abort_flag, limit)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        // the lesser products' other columns have been read: the wait above was for a
                        // later drain than theirs
                        if (drains++ == LESSER) {
                            small ^= (tmem + 256) ^ (tmem + 384);
                            drains = 1;
                            begun = false;
                        }
                    }
                    const uint32_t d = F32 ? tmem + acc * 128 : tmem;
                    for (int kb = k0; kb < k1 && ok; ++kb) {
                        if (!F32 && blocks++ == LONG) {
                            if (issue) mma_commit(tfull_bar(0));
                            if (!warp_wait(tempty_bar(0), acc_phase, abort_flag, limit)) {
                                ok = false;
                                break;
                            }
                            tc_fence_after();
                            acc_phase ^= 1u;
                            blocks = 1;
                            begun = false;
                        }
                        int at[S::PARTS] = {};  // the parts' slots
                        auto product = [&](int pa, int pb, uint32_t dst, bool fresh) {
                            const uint64_t as = wa + static_cast<uint32_t>(at[pa] * (slot_bytes >> 4));
                            const uint64_t bs = wb + static_cast<uint32_t>(at[pb] * (slot_bytes >> 4));
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if (issue)
                                    mma_f16(dst, as + k * slice_step(a_mn.value), bs + k * slice_step(b_mn.value), id,
                                            fresh && k == 0 ? 0u : 1u);
                        };
#pragma unroll
                        for (int p = 0; p < S::PARTS; ++p) {
                            if (!warp_wait(full_bar(slot), phase, abort_flag, limit)) {
                                ok = false;
                                break;
                            }
                            tc_fence_after();
                            at[p] = slot;
                            if (++slot == g.slots) {
                                slot = 0;
                                phase ^= 1u;
                            }
                            if constexpr (F32) {
                                if (p == 0) {
                                    product(0, 0, d, kb == k0);
                                } else if (p == 1) {
                                    product(1, 1, small, !begun);
                                    product(0, 1, small, false);
                                    product(1, 0, small, false);
                                } else {
                                    product(0, 2, small, false);
                                    product(2, 0, small, false);
                                }
                            } else {
                                product(0, 0, d, !begun);
                            }
                        }
                        if (!ok) break;
                        begun = true;
#pragma unroll
                        for (int p = 0; p < S::PARTS; ++p)
                            if (issue) mma_commit(empty_bar(at[p]));
                    }
                    if (F32 && ok) {
                        if (issue) mma_commit(tfull_bar(acc));
                        if (++acc == 2) {
                            acc = 0;
                            acc_phase ^= 1u;
                        }
                    }
                }
            });
        }
        if (!F32 && ok && issue) mma_commit(tfull_bar(0));
        if (issue) mma_commit(drain_bar);
        const long long t0 = clock64();
        while (!mbar_test(drain_bar, 0) && clock64() - t0 < WAIT_CYCLES) {
        }
    } else {
        const int quarter = warp & 3;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        const int row = quarter * 32 + lane;
        // the row's 16-byte unit u of the CTA's binary32 tile: units swapped by
        // row, so that 32 rows' stores of one unit meet different banks
        auto put = [&](int c, const float (&v)[32]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t at = base + row * 512 + (((c / 4 + j) ^ lane) << 4);
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v[4 * j]), "f"(v[4 * j + 1]),
                             "f"(v[4 * j + 2]), "f"(v[4 * j + 3])
                             : "memory");
            }
        };
        auto ready = [&](int acc, uint32_t phase) {
            int r = 0;
            if (lane == 0) r = mbar_wait(tfull_bar(acc), phase, abort_flag, limit) ? 1 : 0;
            r = __shfl_sync(0xffffffffu, r, 0);
            tc_fence_after();
            return r != 0;
        };
        const bool rows_here = mt * 128 + quarter * 32 < g.M;
        if constexpr (F32) {
            float sum[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < 32; ++i) sum[c][i] = 0.0f;
            int acc = 0, lesser = 0, since = 0;
            uint32_t phase = 0;
            auto add = [&](uint32_t from) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t r[32];
                    tmem_ld32(from + c * 32, r);
#pragma unroll
                    for (int i = 0; i < 32; ++i) sum[c][i] = __fadd_rn(sum[c][i], __uint_as_float(r[i]));
                }
            };
            int drains = 0;  // as the MMA warp's loops make them
            for (int seg = 0; seg < g.segments; ++seg) {
                int lo, hi;
                part(seg, lo, hi);
                drains += (hi - lo + CHUNK - 1) / CHUNK;
            }
            for (int u = 0; u < drains; ++u) {
                if (since++ == LESSER) {
                    add(lanes + 256 + lesser * 128);
                    lesser ^= 1;
                    since = 1;
                }
                if (!ready(acc, phase)) {
                    done = false;
                    break;
                }
                add(lanes + acc * 128);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty_bar(acc));
                if (++acc == 2) {
                    acc = 0;
                    phase ^= 1u;
                }
            }
            if (done && rows_here) {
                add(lanes + 256 + lesser * 128);
#pragma unroll
                for (int c = 0; c < 4; ++c) put(c * 32, sum[c]);
            }
        } else {
            for (int u = 0; u < sums; ++u) {
                done = ready(0, u & 1);
                if (!done) break;
                if (sums > 1) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) tmem_add32(lanes + 128 + c * 32, lanes + c * 32, u == 0);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tempty_bar(0));
                }
            }
            if (done && rows_here) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t r[32];
                    float v[32];
                    tmem_ld32(lanes + (sums > 1 ? 128 : 0) + c * 32, r);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
                    put(c * 32, v);
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    // all of the cluster's tiles are in shared memory
    if (g.splits > 1) cluster_arrive_wait();
    else __syncthreads();
    tc_fence_after();
    // a tile is whole if no CTA of the cluster gave up: the others' sums lack its part
    bool gave_up = *abort_flag != 0;
    if (g.splits > 1) {
        const uint32_t flag = bars + 8u * (2 * S::MAX_SLOTS + 5) + 4;
        gave_up = __any_sync(0xffffffffu, ld_cluster1(map_to_rank(flag, lane < g.splits ? lane : 0)));
    }
    if (!gave_up) {
        const int rows = min(128, g.M - mt * 128);
        const int64_t row0 = static_cast<int64_t>(mt) * 128, col0 = static_cast<int64_t>(nt) * BN;
        const float scale = scale_of<T>(g.e);
        // 16-byte unit `unit` of row r of the tiles, added over the cluster in rank order, all loads under way together
        auto sum4 = [&](int r, int unit) {
            const uint32_t at = r * 512 + ((unit ^ (r & 31)) << 4);
            if (g.splits == 1) return lds4(base + at);
            float4 q[MAX_SPLIT];
#pragma unroll
            for (int s = 0; s < MAX_SPLIT; ++s)
                if (s < g.splits) q[s] = ld_cluster(map_to_rank(base, s) + at);
            float4 t = q[0];
#pragma unroll
            for (int s = 1; s < MAX_SPLIT; ++s)
                if (s < g.splits) {
                    t.x = __fadd_rn(t.x, q[s].x);
                    t.y = __fadd_rn(t.y, q[s].y);
                    t.z = __fadd_rn(t.z, q[s].z);
                    t.w = __fadd_rn(t.w, q[s].w);
                }
            return t;
        };
        if (g.e.vec == 1) {
            // 8 columns a thread, always the same ones
            constexpr int UNITS = BN / 8;
            static_assert(THREADS % UNITS == 0, "a thread keeps its columns");
            const int id = rank * THREADS + static_cast<int>(threadIdx.x);
            const int c = id % UNITS * 8;
            if (col0 + c < g.N) {
                float bias[DUAL ? 2 : 1][8];
                bias8<T, DUAL>(g.e, col0 + c, bias);
#pragma unroll(DUAL ? 1 : 2)
                for (int r = id / UNITS; r < rows; r += g.splits * (THREADS / UNITS)) {
                    float z[8], u[8];
                    auto sum = [&](int unit, float (&v)[8]) {
                        const float4 lo = sum4(r, unit), hi = sum4(r, unit + 1);
                        v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
                        v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
                    };
                    sum(c / 4, z);
                    if constexpr (DUAL) sum(16 + c / 4, u);
                    finish8<T, DUAL>(g.e, row0 + r, col0 + c, bias, z, u, scale);
                }
            }
        } else {
            // rows off 16 bytes: a warp a row, every 32nd column (or pair of them) a lane,
            // ROWS rows together
            constexpr int STEPS = BN / 32, ROWS = 4, WARPS = THREADS / 32, ALL = ROWS * STEPS;
            const Epilogue& e = g.e;
            const int step = g.splits * WARPS;
            auto rows_of = [&](auto pairs) {
                constexpr bool P = pairs.value;
                // element k of the ROWS rows: its column, its row, whether it exists, where it is
                auto col = [&](int k) { return P ? k % STEPS / 2 * 64 + lane * 2 + (k & 1) : k % STEPS * 32 + lane; };
                float b0[STEPS], b1[STEPS];
#pragma unroll
                for (int j = 0; j < STEPS; ++j) {
                    const bool in = col0 + col(j) < g.N;
                    b0[j] = in ? bias1<T>(e, 0, col0 + col(j)) : 0.0f;
                    b1[j] = DUAL && in ? bias1<T>(e, 1, col0 + col(j)) : 0.0f;
                }
                for (int r0 = rank * WARPS + warp; r0 < rows; r0 += ROWS * step) {
                    auto row = [&](int k) { return r0 + k / STEPS * step; };
                    auto here = [&](int k) { return row(k) < rows && col0 + col(k) < g.N; };
                    auto at = [&](int k, int64_t ld) { return (row0 + row(k)) * ld + col0 + col(k); };
                    if (g.splits > 1) {  // the cluster's sums of these rows, in place of this CTA's part
#pragma unroll
                        for (int i = 0; i < ROWS; ++i) {
                            const int r = r0 + i * step;
                            if (r >= rows) break;
                            const float4 t = sum4(r, lane);
                            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(
                                             base + r * 512 + ((lane ^ (r & 31)) << 4)),
                                         "f"(t.x), "f"(t.y), "f"(t.z), "f"(t.w)
                                         : "memory");
                        }
                        __syncwarp();
                    }
                    float z[ALL], u[DUAL ? ALL : 1];
                    [[maybe_unused]] float res[DUAL ? 1 : ALL];
                    if constexpr (!DUAL) {
                        if (e.residual && e.y) {
                            const T* from = static_cast<const T*>(e.residual);
#pragma unroll
                            for (int k = 0; k < ALL; k += P ? 2 : 1)
                                if (here(k)) {
                                    if constexpr (P) {
                                        const float2 f = ld2(from + at(k, e.res_ld));
                                        res[k] = f.x;
                                        res[k + 1] = f.y;
                                    } else {
                                        res[k] = ld1(from + at(k, e.res_ld));
                                    }
                                }
                        }
                    }
                    auto tile = [&](int k, int c) {
                        const int r = min(row(k), rows - 1);
                        return __fmul_rn(lds1(base + r * 512 + (((c / 4) ^ (r & 31)) << 4) + (c & 3) * 4), scale);
                    };
#pragma unroll
                    for (int k = 0; k < ALL; ++k) {
                        z[k] = __fadd_rn(tile(k, col(k)), b0[k % STEPS]);
                        if constexpr (DUAL) u[k] = __fadd_rn(tile(k, 64 + col(k)), b1[k % STEPS]);
                    }
                    auto store = [&](void* p, const float* v) {
                        T* to = static_cast<T*>(p);
#pragma unroll
                        for (int k = 0; k < ALL; k += P ? 2 : 1)
                            if (here(k)) {
                                if constexpr (P) st2(to + at(k, e.N), v[k], v[k + 1]);
                                else st1(to + at(k, e.N), v[k]);
                            }
                    };
                    if (e.pre[0]) store(e.pre[0], z);
                    if (DUAL && e.pre[1]) store(e.pre[1], u);
                    if (!e.y) continue;
                    act_all<T>(e.act, z);
                    if constexpr (DUAL) {
#pragma unroll
                        for (int k = 0; k < ALL; ++k) z[k] = __fmul_rn(z[k], u[k]);
                    } else if (e.residual) {
#pragma unroll
                        for (int k = 0; k < ALL; ++k) z[k] = __fadd_rn(z[k], res[k]);
                    }
                    store(e.y, z);
                }
            };
            if (e.vec == 2) rows_of(std::true_type{});
            else rows_of(std::false_type{});
        }
    } else if (threadIdx.x == 0) {
        atomicExch(g.status, QSML_E_TIMEOUT);
    }
    // no CTA leaves while another reads its tile
    if (g.splits > 1) cluster_arrive_wait();
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols) : "memory");
    }
}

// ---------------------------------------------------------------------------
// Large products: persistent pairs of SMs (cta_group::2), the epilogue of a tile
// under the products of the next.
//   binary16: 256 x 256 of the result a pair (dual: 128 columns of each weight, one
//     from each CTA), five slots of 32 KiB a CTA, two accumulators of 256 columns;
//   binary32: 256 x 128 (dual: 64 of each), eight slots of one part (24 KiB a CTA), two
//     accumulators for the drains of the main product and two, in turn, for the lesser
//     ones.
// Each CTA loads its own 128 rows of A and half of the tile's columns of B; the
// leader issues the MMAs of both.  Roles and barriers as in k_linear_tc, the
// leader's full barrier counting both CTAs' bytes.
// ---------------------------------------------------------------------------
template <bool F32> struct PairShape {
    static constexpr int PARTS = F32 ? 3 : 1;
    static constexpr int SLOTS = F32 ? 8 : 5;                 // a tile of A and one of B each, of one part
    static constexpr int EPI = 8;                             // epilogue warps
    static constexpr int THREADS = 64 + 32 * EPI;
    static constexpr int BCOLS = F32 ? 64 : 128;              // columns of B a CTA
    static constexpr int SLOT = TILE_BYTES + BCOLS * 128;
    static constexpr int NACC = 2 * BCOLS;                    // accumulator columns
    static constexpr int OUT_WARP = F32 ? 4096 : 8192;        // epilogue staging of a warp's 32 rows
    static constexpr int OUT = EPI * OUT_WARP;
    static constexpr size_t SMEM = size_t(SLOTS) * SLOT + OUT + 1024 + 256;
    static_assert(SMEM <= 232448, "shared memory");
};
constexpr int PAIR_GROUP_M = 16;  // tiles of 16 row blocks run together: A and B panels stay in L2

__device__ __forceinline__ void mma_f16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
}

template <bool F32, bool DUAL>
__global__ void __launch_bounds__(PairShape<F32>::THREADS, 1) k_linear_pair(const __grid_constant__ TcArgs g) {
    using T = std::conditional_t<F32, float, __half>;
    using S = PairShape<F32>;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char* gbase = smem_raw + (base - raw);
    const uint32_t out_stage = base + S::SLOTS * S::SLOT;
    const uint32_t bars = out_stage + S::OUT;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (S::SLOTS + s); };
    auto tfull_bar = [&](int a) { return bars + 8u * (2 * S::SLOTS + a); };
    auto tempty_bar = [&](int a) { return bars + 8u * (2 * S::SLOTS + 2 + a); };
    auto sempty_bar = [&](int a) { return bars + 8u * (2 * S::SLOTS + 4 + a); };  // binary32: lesser products read
    const uint32_t drain_bar = bars + 8u * (2 * S::SLOTS + 6);
    unsigned char* misc = gbase + S::SLOTS * S::SLOT + S::OUT + 8 * (2 * S::SLOTS + 7);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 4);

    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::SLOTS; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), 2 * S::EPI);  // the epilogue warps of both CTAs
            mbar_init(sempty_bar(a), 2 * S::EPI);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_begin();
    // not the context's limit: copies in flight complete on the other CTA's barrier, so
    // a pair gives up only when something is wrong
    constexpr long long limit = WAIT_CYCLES;

    constexpr int BN = DUAL ? S::BCOLS : 2 * S::BCOLS;  // result columns a tile
    const int total = g.tiles_m * g.tiles_n;
    const int pairs = static_cast<int>(gridDim.x >> 1), pair = static_cast<int>(blockIdx.x >> 1);
    auto decode = [&](int t, int& mt, int& nt) {
        const int group = t / (PAIR_GROUP_M * g.tiles_n);
        const int first = group * PAIR_GROUP_M;
        const int gm = min(PAIR_GROUP_M, g.tiles_m - first);
        const int within = t - first * g.tiles_n;
        mt = first + within % gm;
        nt = within / gm;
    };
    // binary32: drains a tile (the CHUNK k-blocks between them counted by segment)
    const int drains = (g.kb + CHUNK - 1) / CHUNK * g.segments;
    // binary16: accumulators a tile; where there are several, the second one's columns hold their sum
    const int sums = (g.kb * g.segments + LONG - 1) / LONG;
    if (warp == 0) {
        const bool issue = elect_one();
        int slot = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = pair; t < total && ok; t += pairs) {
            int mt, nt;
            decode(t, mt, nt);
            const int row = mt * 256 + static_cast<int>(rank) * 128;
            const int col = DUAL ? nt * BN : nt * BN + static_cast<int>(rank) * S::BCOLS;
            for (int sp = 0; sp < g.segments && ok; ++sp) {
                const int seg = sp / g.halves, half = sp - seg * g.halves;
                const CUtensorMap *ma = &g.a[seg], *mb = &g.b[DUAL ? rank : seg];
                const int ha = g.a_halves ? half : 0, hb = g.b_halves ? half : 0;
                by_order(g.a_mn[seg], g.b_mn[DUAL ? 0 : seg], [&](auto a_mn, auto b_mn) {
                    for (int kb = 0; kb < g.kb && ok; ++kb) {
#pragma unroll
                        for (int p = 0; p < S::PARTS; ++p) {
                            if (!warp_wait(empty_bar(slot), phase ^ 1u, abort_flag, limit)) {
                                ok = false;
                                break;
                            }
                            if (issue && leader) mbar_expect_tx(full_bar(slot), 2 * S::SLOT);
                            const uint32_t bar = map_to_rank(full_bar(slot), 0);
                            const uint32_t at = base + slot * S::SLOT, bt = at + TILE_BYTES;
                            if (issue) {
                                if (a_mn.value) {
                                    tma_load_3d_pair(at, ma, bar, row, kb * 64, F32 ? p : ha);
                                    tma_load_3d_pair(at + 8192, ma, bar, row + 64, kb * 64, F32 ? p : ha);
                                } else {
                                    tma_load_3d_pair(at, ma, bar, kb * 64, row, F32 ? p : ha);
                                }
                                if (b_mn.value) {
#pragma unroll
                                    for (int j = 0; j < S::BCOLS / 64; ++j)
                                        tma_load_3d_pair(bt + j * 8192, mb, bar, col + j * 64, kb * 64, F32 ? p : hb);
                                } else {
                                    tma_load_3d_pair(bt, mb, bar, kb * 64, col, F32 ? p : hb);
                                }
                            }
                            if (++slot == S::SLOTS) {
                                slot = 0;
                                phase ^= 1u;
                            }
                        }
                    }
                });
            }
        }
    } else if (warp == 1) {
        if (leader) {
            const bool issue = elect_one();
            int slot = 0, acc = 0, par = 0;
            uint32_t phase = 0, acc_phase = 0, par_phase = 0;
            bool ok = true;
            auto next_acc = [&]() {
                if (!F32 && sums > 1) {
                    acc_phase ^= 1u;
                } else if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            };
            auto next_par = [&]() {
                if (++par == 2) {
                    par = 0;
                    par_phase ^= 1u;
                }
            };
            for (int t = pair; t < total && ok; t += pairs) {
                if (F32) {
                    if (!warp_wait(sempty_bar(par), par_phase ^ 1u, abort_flag, limit)) break;
                    tc_fence_after();
                }
                uint32_t small = tmem + 256 + par * 128;
                int since = 0;  // binary32: drains of the main product since the lesser ones' last
                if (!F32) {
                    if (!warp_wait(tempty_bar(acc), acc_phase ^ 1u, abort_flag, limit)) break;
                    tc_fence_after();
                }
                bool begun = false;
                int blocks = 0;  // binary16: in the accumulator
                for (int sp = 0; sp < g.segments && ok; ++sp) {
                    const int seg = sp / g.halves;
                    by_order(g.a_mn[seg], g.b_mn[DUAL ? 0 : seg], [&](auto a_mn, auto b_mn) {
                        const uint32_t id = idesc(F32, a_mn.value, b_mn.value, 256, S::NACC);
                        const uint64_t wa = slice_desc(base, a_mn.value, 0), wb = slice_desc(base + TILE_BYTES, b_mn.value, 0);
                        for (int k0 = 0; k0 < g.kb && ok; k0 += F32 ? CHUNK : g.kb) {
                            const int k1 = F32 ? min(k0 + CHUNK, g.kb) : g.kb;
                            if (F32) {
                                if (!warp_wait(tempty_bar(acc), acc_phase ^ 1u, abort_flag, limit)) {
                                    ok = false;
                                    break;
                                }
                                tc_fence_after();
                                if (since++ == LESSER) {  // as at a tile's end
                                    next_par();
                                    if (!warp_wait(sempty_bar(par), par_phase ^ 1u, abort_flag, limit)) {
                                        ok = false;
                                        break;
                                    }
                                    tc_fence_after();
                                    small = tmem + 256 + par * 128;
                                    since = 1;
                                    begun = false;
                                }
                            }
                            const uint32_t d = tmem + acc * S::NACC;
                            for (int kb = k0; kb < k1 && ok; ++kb) {
                                if (!F32 && blocks++ == LONG) {
                                    if (issue) mma_commit_pair(tfull_bar(acc));
                                    next_acc();
                                    if (!warp_wait(tempty_bar(acc), acc_phase ^ 1u, abort_flag, limit)) {
                                        ok = false;
                                        break;
                                    }
                                    tc_fence_after();
                                    blocks = 1;
                                    begun = false;
                                }
                                int at[S::PARTS] = {};  // the parts' slots
                                auto product = [&](int pa, int pb, uint32_t dst, bool fresh) {
                                    const uint64_t as = wa + static_cast<uint32_t>(at[pa] * (S::SLOT >> 4));
                                    const uint64_t bs = wb + static_cast<uint32_t>(at[pb] * (S::SLOT >> 4));
#pragma unroll
                                    for (int k = 0; k < 4; ++k)
                                        if (issue)
                                            mma_f16_pair(dst, as + k * slice_step(a_mn.value), bs + k * slice_step(b_mn.value),
                                                         id, fresh && k == 0 ? 0u : 1u);
                                };
#pragma unroll
                                for (int p = 0; p < S::PARTS; ++p) {
                                    if (!warp_wait(full_bar(slot), phase, abort_flag, limit)) {
                                        ok = false;
                                        break;
                                    }
                                    tc_fence_after();
                                    at[p] = slot;
                                    if (++slot == S::SLOTS) {
                                        slot = 0;
                                        phase ^= 1u;
                                    }
                                    if constexpr (F32) {
                                        if (p == 0) {
                                            product(0, 0, d, kb == k0);
                                        } else if (p == 1) {
                                            product(1, 1, small, !begun);
                                            product(0, 1, small, false);
                                            product(1, 0, small, false);
                                        } else {
                                            product(0, 2, small, false);
                                            product(2, 0, small, false);
                                        }
                                    } else {
                                        product(0, 0, d, !begun);
                                    }
                                }
                                if (!ok) break;
                                begun = true;
#pragma unroll
                                for (int p = 0; p < S::PARTS; ++p)
                                    if (issue) mma_commit_pair(empty_bar(at[p]));
                            }
                            if (F32 && ok) {
                                if (issue) mma_commit_pair(tfull_bar(acc));
                                next_acc();
                            }
                        }
                    });
                }
                if (!ok) break;
                if (!F32) {
                    if (issue) mma_commit_pair(tfull_bar(acc));
                    next_acc();
                }
                next_par();
            }
            if (issue) mma_commit_pair_local(drain_bar);
            const long long t0 = clock64();
            while (!mbar_test(drain_bar, 0) && clock64() - t0 < WAIT_CYCLES) {
            }
        }
    } else {
        const int quarter = warp & 3;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        int acc = 0, par = 0;
        uint32_t phase = 0;
        auto ready = [&]() {
            int r = 0;
            if (lane == 0) r = mbar_wait(tfull_bar(acc), phase, abort_flag, limit) ? 1 : 0;
            r = __shfl_sync(0xffffffffu, r, 0);
            tc_fence_after();
            return r != 0;
        };
        auto release = [&](uint32_t bar) {  // this warp is done with an accumulator
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(map_to_rank(bar, 0));
        };
        auto next_acc = [&]() {
            if (!F32 && sums > 1) {
                phase ^= 1u;
            } else if (++acc == 2) {
                acc = 0;
                phase ^= 1u;
            }
        };
        bool ok = true;
        for (int t = pair; t < total && ok; t += pairs) {
            int mt, nt;
            decode(t, mt, nt);
            const int row0 = mt * 256 + static_cast<int>(rank) * 128 + quarter * 32;  // first of the warp's 32 rows
            const int64_t col0 = static_cast<int64_t>(nt) * BN;
            // two warps a quarter of the rows, each half of the columns (dual: of both weights')
            const uint32_t stage = out_stage + (warp - 2) * S::OUT_WARP;
            const int cbegin = warp >= 6 ? BN / 2 : 0;
            const int cend = static_cast<int>(min(g.N - col0, static_cast<int64_t>(cbegin + BN / 2)));
            if constexpr (F32) {
            constexpr int WORDS = 32;                       // binary32 a staged row
            constexpr int STEP = DUAL ? WORDS / 2 : WORDS;  // result columns a round
            // 16-byte unit j of the lane's row: units swapped by row against bank conflicts
            auto unit_at = [&](int row, int j) {
                return stage + row * (WORDS * 4) + ((j ^ (row & (WORDS / 4 - 1))) << 4);
            };
            auto put = [&](int j, float a, float b, float c, float d) {
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(unit_at(lane, j)), "f"(a), "f"(b), "f"(c),
                             "f"(d)
                             : "memory");
            };
            auto take = [&](int row, int j, float (&v)[8]) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(v[4 * h]), "=f"(v[4 * h + 1]), "=f"(v[4 * h + 2]), "=f"(v[4 * h + 3])
                                 : "r"(unit_at(row, j + h))
                                 : "memory");
            };
            // the staged round's outputs: 8 columns a lane, whole rows of STEP together
            auto finish = [&](int c0) {
                __syncwarp();
                constexpr int UNITS = STEP / 8, ROWS = 32 / UNITS;
                const int un = lane % UNITS;
                const int64_t col = col0 + c0 + un * 8;
                if (col < g.N) {
                    float bias[DUAL ? 2 : 1][8];
                    bias8<T, DUAL>(g.e, col, bias);
#pragma unroll 2
                    for (int r = lane / UNITS; r < 32; r += ROWS) {
                        if (row0 + r >= g.M) break;
                        float z[8], v[8];
                        take(r, un * 2, z);
                        if constexpr (DUAL) take(r, WORDS / 8 + un * 2, v);
                        finish8<T, DUAL>(g.e, row0 + r, col, bias, z, v);
                    }
                }
                __syncwarp();
            };
                // the drains, added in registers: 64 columns of a row a thread, those of
                // the accumulator from `from(c)` on
                auto from = [&](int c) { return DUAL ? (c < 1 ? cbegin : 64 + cbegin) : cbegin + c * 32; };
                float sum[2][32];
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int i = 0; i < 32; ++i) sum[c][i] = 0.0f;
                auto drain = [&](uint32_t d) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t r[32];
                        tmem_ld32(d + from(c), r);
#pragma unroll
                        for (int i = 0; i < 32; ++i) sum[c][i] = __fadd_rn(sum[c][i], __uint_as_float(r[i]));
                    }
                };
                auto drain_lesser = [&]() {
                    drain(lanes + 256 + par * 128);
                    release(sempty_bar(par));
                    par ^= 1;
                };
                for (int u = 0; u < drains; ++u) {
                    if (u > 0 && u % LESSER == 0) drain_lesser();
                    if (!ready()) {
                        ok = false;
                        break;
                    }
                    drain(lanes + acc * 128);
                    release(tempty_bar(acc));
                    next_acc();
                }
                if (!ok) break;
                drain_lesser();
#pragma unroll
                for (int round = 0; round < 2; ++round) {
                    if (cbegin + round * STEP >= cend) break;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        // dual: columns 16 round .. + 15 of both weights', else 32 of one
                        const float* v = DUAL ? &sum[j / 4][round * 16 + (j % 4) * 4] : &sum[round][j * 4];
                        put(j, v[0], v[1], v[2], v[3]);
                    }
                    finish(cbegin + round * STEP);
                }
            } else {
                // registers to binary16 staging to whole row segments: staging costs the
                // shared-memory bandwidth that the operands' loads and reads use up
                constexpr int COLS = DUAL ? 32 : 64;  // a round
                using Rows = HalfRows<COLS>;
                const Rows out{stage}, kept0{stage + Rows::BYTES}, kept1{stage + 2 * Rows::BYTES};
                static_assert((DUAL ? 3 : 2) * Rows::BYTES <= S::OUT_WARP, "staging");
                const int rows = max(0, min(32, g.M - row0));
                const Epilogue& e = g.e;
                const int vec = e.vec;
                // several accumulators: each is added to the second's columns, so that the next
                // tile's products begin under this one's outputs
                const bool joined = sums > 1;
                for (int u = 0; joined && u < sums; ++u) {
                    ok = ready();
                    if (!ok) break;
                    for (int c0 = cbegin; c0 < cend; c0 += 32) {
                        tmem_add32(lanes + S::NACC + c0, lanes + c0, u == 0);
                        if constexpr (DUAL) tmem_add32(lanes + S::NACC + 128 + c0, lanes + 128 + c0, u == 0);
                    }
                    release(tempty_bar(0));
                    next_acc();
                }
                if (!ok || (!joined && !ready())) break;
                const uint32_t d = lanes + (joined ? 1 : acc) * S::NACC;
                auto read = [&]() {
                    if (!joined) release(tempty_bar(acc));
                };
                const float scale = scale_of<T>(e);
                if (cbegin >= cend) read();
                for (int c0 = cbegin; c0 < cend; c0 += COLS) {
                    const int64_t col = col0 + c0;
                    if (!DUAL && e.residual && e.y) {
                        out.template copy<true>(static_cast<__half*>(const_cast<void*>(e.residual)), e.res_ld, col, g.N,
                                                row0, rows, vec);
                        __syncwarp();
                    }
#pragma unroll
                    for (int h = 0; h < COLS / 32; ++h) {
                        if (c0 + h * 32 >= cend) break;
                        float z[32], u[32];
                        auto load = [&](uint32_t from, float (&v)[32]) {
                            uint32_t r[32];
                            tmem_ld32(from, r);
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
                            if (scale != 1.0f) {
#pragma unroll
                                for (int i = 0; i < 32; ++i) v[i] = __fmul_rn(v[i], scale);
                            }
                        };
                        load(d + c0 + h * 32, z);
                        if constexpr (DUAL) load(d + 128 + c0, u);
                        if (c0 + h * 32 + 32 >= cend) read();
                        add_bias32(e, 0, col + h * 32, z);
                        if constexpr (DUAL) add_bias32(e, 1, col, u);
                        if (e.pre[0]) kept0.put(lane, h, z);
                        if constexpr (DUAL) {
                            if (e.pre[1]) kept1.put(lane, h, u);
                        }
                        if (e.y) {
                            act_all<__half>(e.act, z);
                            if constexpr (DUAL) {
#pragma unroll
                                for (int i = 0; i < 32; ++i) z[i] = __fmul_rn(z[i], u[i]);
                            } else if (e.residual) {
                                out.add(lane, h, z);
                            }
                            out.put(lane, h, z);
                        }
                    }
                    __syncwarp();
                    if (e.y) out.template copy<false>(static_cast<__half*>(e.y), g.N, col, g.N, row0, rows, vec);
                    if (e.pre[0]) kept0.template copy<false>(static_cast<__half*>(e.pre[0]), g.N, col, g.N, row0, rows, vec);
                    if (DUAL && e.pre[1])
                        kept1.template copy<false>(static_cast<__half*>(e.pre[1]), g.N, col, g.N, row0, rows, vec);
                    __syncwarp();
                }
                if (!joined) next_acc();
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        if (threadIdx.x == 0) atomicExch(g.status, QSML_E_TIMEOUT);
        // copies still in flight complete on the leader's barrier: give them time
        // to land before the pair's shared memory is released
        const long long t0 = clock64();
        while (clock64() - t0 < 20000000LL) {
        }
    }
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---------------------------------------------------------------------------
// Operands for TMA
// ---------------------------------------------------------------------------

// A copy to 16-bit rows of `pitch`: binary16 as it is, binary32 as its three bf16
// parts (`plane` elements apart); `outer` rows of `inner` from any strides.
struct StageJob {
    const void* src;
    uint16_t* dst;
    int64_t outer, inner, os, is, pitch, plane;
    int64_t first;  // block of the launch that begins it
    int vec;        // 16-byte aligned rows of unit stride
};
constexpr int MAX_JOBS = 8;
struct StageJobs {
    StageJob job[MAX_JOBS];
    int n = 0;
    int64_t blocks = 0;
};

// Eight consecutive elements of the stored order a thread.  Bound by HBM: binary32
// reads 4 and writes 6 bytes an element.
template <typename T> __global__ void __launch_bounds__(256) k_linear_stage(const __grid_constant__ StageJobs jobs) {
    pdl_begin();
    int k = 0;
    while (k + 1 < jobs.n && static_cast<int64_t>(blockIdx.x) >= jobs.job[k + 1].first) ++k;
    const StageJob& j = jobs.job[k];
    const int64_t groups = (j.inner + 7) / 8, total = j.outer * groups;
    const int64_t blocks = (k + 1 < jobs.n ? jobs.job[k + 1].first : jobs.blocks) - j.first;
    for (int64_t i = (blockIdx.x - j.first) * 256 + threadIdx.x; i < total; i += blocks * 256) {
        const int64_t o = i / groups, c = (i - o * groups) * 8;
        const int n = j.inner - c < 8 ? static_cast<int>(j.inner - c) : 8;
        const T* p = static_cast<const T*>(j.src) + o * j.os + c * j.is;
        float v[8];
        if (j.vec && n == 8) {
            ldg8(p, 8, true, v);
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = q < n ? ld1(p + q * j.is) : 0.0f;
        }
        uint16_t* d = j.dst + o * j.pitch + c;
        if constexpr (sizeof(T) == 2) store8(reinterpret_cast<__half*>(d), 8, true, v);
        else split8(v, d, j.plane);
    }
}

struct Staged {
    const void* p = nullptr;
    int64_t inner = 0, outer = 0, pitch = 0, plane = 0;  // 16-bit elements
    bool trans = false;  // stored as the matrix's transpose
};

// The matrix as TMA will read it; a copy, where there has to be one, is added to
// `jobs`.  want: 0 rows, 1 columns contiguous, -1 as it lies.
qsml_status_t stage(Context* ctx, Workspace& ws, StageJobs* jobs, const Mat& m, bool f32, int want, Staged* s) {
    const bool by_rows = m.cs == 1 || m.cols == 1, by_cols = m.rs == 1 || m.rows == 1;
    s->trans = want >= 0 ? want == 1 : !by_rows && by_cols;
    s->inner = s->trans ? m.rows : m.cols;
    s->outer = s->trans ? m.cols : m.rows;
    int64_t os = s->trans ? m.cs : m.rs, is = s->trans ? m.rs : m.cs;
    if (s->inner == 1) is = 1;
    if (s->outer == 1) os = line_pitch(s->inner);
    s->p = m.p;
    s->pitch = os;
    s->plane = m.plane;
    if (m.plane) return QSML_OK;
    const int es = f32 ? 4 : 2;
    if (!f32 && is == 1 && aligned16(m.p) && os % 8 == 0 && os >= s->inner && os < (int64_t(1) << 38)) return QSML_OK;
    StageJob& j = jobs->job[jobs->n];
    j.src = m.p;
    j.outer = s->outer;
    j.inner = s->inner;
    j.os = os;
    j.is = is;
    j.pitch = line_pitch(s->inner);
    j.plane = j.pitch * s->outer;
    j.vec = is == 1 && aligned16(m.p) && (os * es) % 16 == 0;
    void* dst = nullptr;
    QSML_TRY_STATUS(ws.get(static_cast<size_t>(j.plane) * 2 * (f32 ? 3 : 1), &dst));
    j.dst = static_cast<uint16_t*>(dst);
    j.first = jobs->blocks;
    int64_t blocks = (s->outer * ((s->inner + 7) / 8) + 255) / 256;
    if (blocks > int64_t(ctx->num_sms) * 16) blocks = int64_t(ctx->num_sms) * 16;
    jobs->blocks += blocks;
    ++jobs->n;
    s->p = dst;
    s->pitch = j.pitch;
    s->plane = f32 ? j.plane : 0;
    return QSML_OK;
}

qsml_status_t run_jobs(Context* ctx, const StageJobs& jobs, bool f32) {
    if (jobs.n == 0) return QSML_OK;
    const cudaError_t e = launch_pdl(f32 ? k_linear_stage<float> : k_linear_stage<__half>,
                                     dim3(static_cast<unsigned>(jobs.blocks)), dim3(256), 0, ctx->stream, jobs);
    if (e != cudaSuccess) return check_cuda(ctx, e, "k_linear_stage");
    return after_launch(ctx, "k_linear_stage");
}

// mn: MN-major boxes of 64 x 64 k, else K-major boxes of 64 k x `rows`.
bool operand_map(CUtensorMap* map, const Staged& s, bool f32, bool mn, uint32_t rows) {
    const uint64_t planes = f32 ? 3 : s.plane ? 2 : 1;
    return make_map(map, s.p, s.inner, s.outer, planes, s.pitch * 2, (s.plane ? s.plane : s.pitch * s.outer) * 2, 64,
                    mn ? 64 : rows, f32 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
}

// Pairs of SMs that the device holds at once (0: none), once per device and kernel.
template <bool F32, bool DUAL> qsml_status_t max_pairs(Context* ctx, int* pairs) {
    static std::mutex mu;
    static int known[64] = {};
    std::lock_guard<std::mutex> lk(mu);
    int& n = known[ctx->device & 63];
    if (n == 0) {
        auto kernel = k_linear_pair<F32, DUAL>;
        QSML_TRY_STATUS(check_cuda(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                             static_cast<int>(PairShape<F32>::SMEM)),
                                   "linear: shared-memory attribute"));
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.gridDim = dim3(2 * (ctx->num_sms / 2));
        cfg.blockDim = dim3(PairShape<F32>::THREADS);
        cfg.dynamicSmemBytes = PairShape<F32>::SMEM;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            n = -1;
        }
    }
    *pairs = n < 0 ? 0 : n;
    return QSML_OK;
}

template <bool F32, bool DUAL> qsml_status_t launch_pair(Context* ctx, const Problem& p, TcArgs& g, int pairs) {
    using S = PairShape<F32>;
    constexpr int BN = DUAL ? S::BCOLS : 2 * S::BCOLS;
    g.tiles_m = static_cast<int>((p.M + 255) / 256);
    g.tiles_n = static_cast<int>((p.N + BN - 1) / BN);
    g.splits = 1;
    const int64_t tiles = static_cast<int64_t>(g.tiles_m) * g.tiles_n;
    if (tiles > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "linear: too many output tiles");
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(2 * (tiles < pairs ? tiles : pairs)));
    cfg.blockDim = dim3(S::THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = ctx->stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const char* name = F32 ? "k_linear_pair<f32>" : "k_linear_pair<f16>";
    const cudaError_t e = cudaLaunchKernelEx(&cfg, k_linear_pair<F32, DUAL>, g);
    if (e != cudaSuccess) return check_cuda(ctx, e, name);
    return after_launch(ctx, name);
}

// Asks for the kernel's shared memory, once a device.
template <bool F32, bool DUAL, int NP> qsml_status_t opt_in(Context* ctx) {
    static std::mutex mu;
    static uint64_t done = 0;
    std::lock_guard<std::mutex> lk(mu);
    const uint64_t bit = uint64_t(1) << (ctx->device & 63);
    if (done & bit) return QSML_OK;
    using S = Shape<F32>;
    QSML_TRY_STATUS(check_cuda(ctx, cudaFuncSetAttribute(k_linear_tc<F32, DUAL, NP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                         static_cast<int>(S::smem(S::DEEP_RING))),
                               "linear: shared-memory attribute"));
    done |= bit;
    return QSML_OK;
}

// few rows: slots are small, and with the small ring the next call's CTAs fit beside
// this one's, so that their set-up overlaps its end (gated 5 x 4096 x 11008 35.9 ->
// 31.5 us; asking for the weight's first blocks ahead of the wait, into L2, took 36)
template <bool F32> int ring_bytes(Context* ctx, int64_t ctas, bool whole) {
    return ctas <= ctx->num_sms && whole ? Shape<F32>::DEEP_RING : Shape<F32>::RING;
}

// CTAs that share a tile's sum.
// One row of tiles: every operand of weight is read once, HBM bounds the whole, and
// as many as the device holds at once pull it fastest (a second turn costs: the gated
// 5 x 4096 x 11008 took 35 us unsplit in one turn and 41 us in three parts and two).
// More rows: the tensor pipe of a SM bounds.  A SM works off its CTAs' k-blocks, and
// each turn has about OVER blocks' time of beginning and end, a joint sum half of it
// again; the fewest such blocks win, fewer splits on a tie (512 x 11008 x 4096, 128
// tiles: 45 us unsplit, 49 in two; 256 x 11008 x 4096, 64 tiles: 41 us unsplit, 29 in
// two, 37 in three; binary32 128 x 8192 x 1024, 8 tiles of one row: 139 us unsplit, 52 in
// four, 39 in eight).
// The cost of products in one launch is reckoned as if all had the longest sum.
struct Split {
    int64_t tiles, blocks;
    int64_t most;  // splits at most
    bool one_row;
    bool whole;    // operand tiles of A of 128 rows
    int splits = 1;
    int64_t cost = INT64_MAX;
};
template <bool F32, bool DUAL> qsml_status_t best_split(Context* ctx, Split* w) {
    using S = Shape<F32>;
    QSML_TRY_STATUS((opt_in<F32, DUAL, 1>(ctx)));  // the occupancy below counts on it
    static std::mutex mu;
    // clusters of each size that the device holds, with the small ring and the deep one
    static int held[64][2][MAX_SPLIT + 1] = {};
    std::lock_guard<std::mutex> lk(mu);
    constexpr int64_t OVER = F32 ? 2 : 8;
    for (int s = 1; s <= MAX_SPLIT && s <= w->most; ++s) {
        const int ring = ring_bytes<F32>(ctx, w->tiles * s, w->whole);
        int& n = held[ctx->device & 63][ring == S::RING ? 0 : 1][s];
        if (n == 0) {
            cudaLaunchConfig_t cfg = {};
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = s;
            attr[0].val.clusterDim.y = 1;
            attr[0].val.clusterDim.z = 1;
            cfg.gridDim = dim3(static_cast<unsigned>(s * ctx->num_sms));
            cfg.blockDim = dim3(THREADS);
            cfg.dynamicSmemBytes = S::smem(ring);
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&n, k_linear_tc<F32, DUAL, 1>, &cfg) != cudaSuccess || n <= 0) {
                cudaGetLastError();
                n = s == 1 ? ctx->num_sms : -1;
            }
        }
        if (n < 0) continue;
        const int64_t turns = (w->tiles + n - 1) / n;
        if (w->one_row) {
            if (turns == 1 && w->blocks >= 2 * s) w->splits = s;
            continue;
        }
        // clusters do not fill every SM: 36 of four take two turns (256 x 8192 x 2304, 27 us;
        // 36 of three 17)
        const int64_t on_a_sm = std::max((w->tiles * s + ctx->num_sms - 1) / ctx->num_sms, turns);
        const int64_t cost = on_a_sm * ((w->blocks + s - 1) / s) + OVER * turns + (s > 1 ? OVER / 2 : 0);
        if (cost < w->cost) {
            w->cost = cost;
            w->splits = s;
        }
    }
    return QSML_OK;
}

inline int64_t tiles_of(const TcArgs& g) { return static_cast<int64_t>(g.tiles_m) * g.tiles_n; }
Split whole_split(const TcArgs& g) {
    const int64_t blocks = static_cast<int64_t>(g.kb) * g.segments;
    return Split{tiles_of(g), blocks, blocks, g.tiles_m == 1, g.a_bytes == TILE_BYTES};
}

template <bool F32, bool DUAL, int NP> qsml_status_t launch(Context* ctx, TcBatch<NP>& all, int splits) {
    using S = Shape<F32>;
    auto kernel = k_linear_tc<F32, DUAL, NP>;
    QSML_TRY_STATUS((opt_in<F32, DUAL, NP>(ctx)));
    int64_t ctas = 0;
    bool whole = true;
    for (int i = 0; i < NP; ++i) {
        all.first[i] = static_cast<int>(ctas);
        ctas += tiles_of(all.g[i]) * splits;
        whole = whole && all.g[i].a_bytes == TILE_BYTES;
        if (ctas > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "linear: too many output tiles");
    }
    const int ring = ring_bytes<F32>(ctx, ctas, whole);
    for (TcArgs& g : all.g) {
        g.splits = splits;
        g.ring = ring;
        g.slots = ring / (g.a_bytes + TILE_BYTES);
        if (g.slots > S::MAX_SLOTS) g.slots = S::MAX_SLOTS;
    }

    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = S::smem(ring);
    cfg.stream = ctx->stream;
    cfg.attrs = attr;
    cfg.numAttrs = splits > 1 ? 2 : 1;
    const char* name = F32 ? "k_linear_tc<f32>" : "k_linear_tc<f16>";
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, all);
    if (e != cudaSuccess) return check_cuda(ctx, e, name);
    return after_launch(ctx, name);
}

template <bool F32, bool DUAL> qsml_status_t launch_one(Context* ctx, const TcArgs& g) {
    Split w = whole_split(g);
    QSML_TRY_STATUS((best_split<F32, DUAL>(ctx, &w)));
    TcBatch<1> all;
    all.g[0] = g;
    return launch<F32, DUAL, 1>(ctx, all, w.splits);
}

// Products in one launch where that is reckoned to take less than one after another:
// each alone splits its sums to fill the GPU, and has a beginning and an end of its own,
// which cost about ALONE blocks' time (backward 512 x 1024 x 1024, binary16, gelu: 25 us
// in two launches, 17 in one; with two weights 2048 x 512 x 512: 33 and 21; binary32 777 x
// 1024 x 1000: 45 and 35; but binary16 8192 x 256 x 512, with sums of 8 and of 128
// blocks: 33 and 37; with two weights 1024 x 1024 x 1024, more CTAs than SMs: 33 and 35).
// `apart`: the cost of the launches it replaces, but for ALONE.
template <bool F32, int NP>
qsml_status_t launch_together(Context* ctx, const TcArgs* const (&g)[NP], int64_t apart, bool* launched) {
    constexpr int64_t ALONE = F32 ? 6 : 24;
    Split all{0, 0, INT64_MAX, false, true};
    for (const TcArgs* one : g) {
        const Split w = whole_split(*one);
        all.tiles += w.tiles;
        all.blocks = std::max(all.blocks, w.blocks);
        all.most = std::min(all.most, w.blocks);
        all.whole = all.whole && w.whole;
    }
    QSML_TRY_STATUS((best_split<F32, false>(ctx, &all)));
    *launched = all.cost < apart + ALONE;
    if (!*launched) return QSML_OK;
    TcBatch<NP> batch;
    for (int i = 0; i < NP; ++i) batch.g[i] = *g[i];
    return launch<F32, false, NP>(ctx, batch, all.splits);
}

// A problem whose operands are known to TMA.
struct Ready {
    Staged a[2], b[2];
    bool pair = false;
    int pairs = 0;
};

qsml_status_t prepare(Context* ctx, Workspace& ws, StageJobs* jobs, const Problem& p, bool f32, Ready* r) {
    // pairs of SMs where the tiles fill at least 60 % of them, else 128 x 128 tiles and
    // split sums (at 64 of 74 pairs, 1024 x 4096 x 4096 takes 27 us against 31; at 32,
    // 512 x 11008 x 4096 57 against 45), unless there are more of those than SMs (160
    // against 40 pairs' tiles, 512 x 4096 x 5000: 44 us against 28; gated 256 x 2048 x
    // 5632: 31 against 18)
    if (f32) QSML_TRY_STATUS((p.dual ? max_pairs<true, true>(ctx, &r->pairs) : max_pairs<true, false>(ctx, &r->pairs)));
    else QSML_TRY_STATUS((p.dual ? max_pairs<false, true>(ctx, &r->pairs) : max_pairs<false, false>(ctx, &r->pairs)));
    const int64_t bn = (f32 ? 128 : 256) / (p.dual ? 2 : 1);
    const int64_t tiles = ((p.M + 255) / 256) * ((p.N + bn - 1) / bn);
    const int64_t small = ((p.M + 127) / 128) * ((p.N + (p.dual ? 63 : 127)) / (p.dual ? 64 : 128));
    r->pair = r->pairs > 0 && p.M > 128 && (tiles * 10 >= r->pairs * 6 || small > ctx->num_sms);
    for (int i = 0; i < p.segments; ++i) QSML_TRY_STATUS(stage(ctx, ws, jobs, p.a[i], f32, -1, &r->a[i]));
    // a dual product's weights share an order: they meet in one MMA
    for (int i = 0; i < (p.dual ? 2 : p.segments); ++i)
        QSML_TRY_STATUS(stage(ctx, ws, jobs, p.b[i], f32, p.dual && i ? (r->b[0].trans ? 1 : 0) : -1, &r->b[i]));
    return QSML_OK;
}

// A problem's arguments; the splits and the ring are the launch's.
qsml_status_t arguments(Context* ctx, const Problem& p, bool f32, const Ready& r, TcArgs* out) {
    TcArgs& g = *out;
    g.e = p.e;
    g.M = static_cast<int>(p.M);
    g.N = static_cast<int>(p.N);
    g.kb = static_cast<int>((p.K + 63) / 64);
    g.tiles_m = static_cast<int>((p.M + 127) / 128);
    g.tiles_n = static_cast<int>((p.N + (p.dual ? 63 : 127)) / (p.dual ? 64 : 128));
    const int na = p.segments, nb = p.dual ? 2 : p.segments;
    g.a_halves = !f32 && r.a[0].plane ? 1 : 0;
    g.b_halves = !f32 && r.b[0].plane ? 1 : 0;
    g.halves = g.a_halves || g.b_halves ? 2 : 1;
    g.segments = p.segments * g.halves;
    g.status = ctx->status;
    // few rows: a K-major tile of A holds no more than them, in whole groups of 8
    int a_rows = !r.pair && p.M <= 64 ? static_cast<int>((p.M + 7) / 8 * 8) : 128;
    for (int i = 0; i < na; ++i)
        if (r.a[i].trans) a_rows = 128;
    g.a_bytes = a_rows * 128;
    const uint32_t b_rows = r.pair ? (f32 ? 64 : 128) : (p.dual ? 64 : 128);  // of a K-major box
    bool ok = true;
    for (int i = 0; i < 2; ++i) {
        const Staged &a = r.a[i < na ? i : 0], &b = r.b[i < nb ? i : 0];
        g.a_mn[i] = a.trans ? 1 : 0;  // stored [K, M]
        g.b_mn[i] = b.trans ? 0 : 1;  // stored [K, N]
        if (i < na) ok = ok && operand_map(&g.a[i], a, f32, g.a_mn[i], static_cast<uint32_t>(a_rows));
        else g.a[i] = g.a[0];
        if (i < nb) ok = ok && operand_map(&g.b[i], b, f32, g.b_mn[i], b_rows);
        else g.b[i] = g.b[0];
    }
    return ok ? QSML_OK : set_error(ctx, QSML_E_CUDA, "linear: tensor map creation failed");
}

qsml_status_t run_one(Context* ctx, const Problem& p, bool f32, const Ready& r, TcArgs& g) {
    if (r.pair) {
        if (f32) return p.dual ? launch_pair<true, true>(ctx, p, g, r.pairs) : launch_pair<true, false>(ctx, p, g, r.pairs);
        return p.dual ? launch_pair<false, true>(ctx, p, g, r.pairs) : launch_pair<false, false>(ctx, p, g, r.pairs);
    }
    if (f32) return p.dual ? launch_one<true, true>(ctx, g) : launch_one<true, false>(ctx, g);
    return p.dual ? launch_one<false, true>(ctx, g) : launch_one<false, false>(ctx, g);
}

// The two products of a backward pass, neither by pairs of SMs.  So the weights are small
// (44 of the pairs' tiles), and HBM does not bound one row of tiles.
template <bool F32>
qsml_status_t run_together(Context* ctx, const Problem* const* p, const Ready* r, const TcArgs* g, bool* launched) {
    Split a = whole_split(g[0]), b = whole_split(g[1]);
    a.one_row = b.one_row = false;
    QSML_TRY_STATUS((best_split<F32, false>(ctx, &a)));
    if (!p[1]->dual) {
        QSML_TRY_STATUS((best_split<F32, false>(ctx, &b)));
        return launch_together<F32, 2>(ctx, {&g[0], &g[1]}, a.cost + b.cost, launched);
    }
    // the gradients of two weights, as two products
    QSML_TRY_STATUS((best_split<F32, true>(ctx, &b)));
    TcArgs w[2];
    for (int i = 0; i < 2; ++i) {
        Problem q = *p[1];
        Ready rq = r[1];
        q.dual = false;
        q.b[0] = p[1]->b[i];
        rq.b[0] = r[1].b[i];
        q.e.y = p[1]->e.pre[i];
        q.e.pre[0] = q.e.pre[1] = nullptr;
        QSML_TRY_STATUS(arguments(ctx, q, F32, rq, &w[i]));
    }
    return launch_together<F32, 3>(ctx, {&g[0], &w[0], &w[1]}, a.cost + b.cost, launched);
}

}  // namespace

qsml_status_t run_tc(Context* ctx, const Problem* const* p, int n, bool f32) {
    Workspace ws(ctx);
    StageJobs jobs;
    Ready r[2];
    TcArgs g[2];
    bool together = n == 2;
    for (int i = 0; i < n; ++i) {
        QSML_TRY_STATUS(prepare(ctx, ws, &jobs, *p[i], f32, &r[i]));
        QSML_TRY_STATUS(arguments(ctx, *p[i], f32, r[i], &g[i]));
        together = together && !r[i].pair;
    }
    QSML_TRY_STATUS(run_jobs(ctx, jobs, f32));
    if (together) {
        bool launched = false;
        QSML_TRY_STATUS(f32 ? run_together<true>(ctx, p, r, g, &launched) : run_together<false>(ctx, p, r, g, &launched));
        if (launched) return QSML_OK;
    }
    for (int i = 0; i < n; ++i) QSML_TRY_STATUS(run_one(ctx, *p[i], f32, r[i], g[i]));
    return QSML_OK;
}

}  // namespace linear
}  // namespace qsml
