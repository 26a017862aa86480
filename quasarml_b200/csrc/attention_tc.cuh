// What the tensor cores' attention kernels share: tiles of 128 tokens of a head by TMA, and
// products of them.
//
// A tile is DP / 64 boxes of 128 rows x 64 columns (128 bytes a row, 128-byte swizzle, columns
// past D zero).  The same tile serves as a K-major operand (its columns summed over: scores) and
// as an MN-major one (its tokens summed over: what is multiplied by P or dS), which come as the
// A operand from TMEM, where the threads that compute them leave them as pairs of binary16.
#pragma once

#include <algorithm>

#include "attention.cuh"
#include "packed.cuh"
#include "tcgen05.cuh"

namespace qsml {
namespace attn {

using namespace tc;

constexpr int TILE = 128;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int DP> struct TileOf {
    static constexpr int BOX = TILE * 128, BOXES = DP / 64, BYTES = BOX * BOXES;
};

// A view's tensor map {columns, tokens, heads, sequences} and which of the last two it moves along.
struct HeadMap {
    CUtensorMap map;
    int sh, sb;
};

inline bool mappable(const View& v, int D, int S, int H, int B) {
    const int64_t most = int64_t(1) << 39;
    auto ok = [&](int64_t s, int64_t n) { return n == 1 || (s >= 0 && s * 2 < most); };
    return D % 8 == 0 && D <= 128 && heads::rows_on(v, 2, 16) && ok(v.s, S) && ok(v.h, H) && ok(v.b, B) && (S == 1 || v.s > 0);
}

inline bool make_head_map(HeadMap* m, const View& v, int D, int S, int H, int B) {
    auto fn = encode_fn();
    if (!fn) return false;
    // a dim that is not moved along has extent 1
    m->sh = H > 1 && v.h > 0;
    m->sb = B > 1 && v.b > 0;
    const cuuint64_t row = static_cast<cuuint64_t>(D) * 2;
    cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(S), m->sh ? static_cast<cuuint64_t>(H) : 1,
                          m->sb ? static_cast<cuuint64_t>(B) : 1};
    cuuint64_t strides[3] = {S > 1 ? static_cast<cuuint64_t>(v.s) * 2 : row, m->sh ? static_cast<cuuint64_t>(v.h) * 2 : row,
                             m->sb ? static_cast<cuuint64_t>(v.b) * 2 : row};
    cuuint32_t box[4] = {64, TILE, 1, 1}, step[4] = {1, 1, 1, 1};
    return fn(&m->map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, v.p, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows [row, row + 128) of head h of sequence b.
template <int DP> __device__ __forceinline__ void load_tile(uint32_t dst, const HeadMap& m, uint32_t bar, int row, int h, int b) {
#pragma unroll
    for (int i = 0; i < DP / 64; ++i)
        asm volatile(
            "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
            ::"r"(dst + i * TileOf<DP>::BOX), "l"(reinterpret_cast<uint64_t>(&m.map)), "r"(i * 64), "r"(row), "r"(m.sh ? h : 0), "r"(m.sb ? b : 0),
            "r"(bar)
            : "memory");
}

// Rows of a landed tile that are not tokens of [0, sink) or [lo, hi) become zeros (a row's 128
// bytes lie together whatever the swizzle); by one warp.
template <int DP> __device__ __forceinline__ void clear_rows(uint32_t tile, int row0, int sink, int lo, int hi) {
    for (int r = threadIdx.x & 31; r < TILE; r += 32) {
        const int row = row0 + r;
        if (row < hi && (row >= lo || row < sink)) continue;
#pragma unroll
        for (int i = 0; i < 8 * (DP / 64); ++i) {
            const uint32_t a = tile + (i >> 3) * TileOf<DP>::BOX + r * 128 + ((i + r) & 7) * 16;  // lanes in different banks
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(0) : "memory");
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}

// binary16 x binary16 -> binary32, M = 128: both operands K-major (scores), or B
// MN-major with N = DP (sums over tokens).
template <int N> constexpr uint32_t IDESC_SCORES = (1u << 4) | (uint32_t(N >> 3) << 17) | (uint32_t(TILE >> 4) << 24);
template <int DP> constexpr uint32_t IDESC_SUMS = (1u << 4) | (1u << 16) | (uint32_t(DP >> 3) << 17) | (uint32_t(TILE >> 4) << 24);

// A descriptor moved on by `bytes`: its address field stays below 2^14 in 16 bytes.
__device__ __forceinline__ uint64_t desc_on(uint64_t d, uint32_t bytes) { return d + (bytes >> 4); }
// A tile as operand of scores (columns summed over) and of sums (tokens summed over).
__device__ __forceinline__ uint64_t score_desc(uint32_t tile) { return smem_desc(tile, 16, 1024); }
template <int DP> __device__ __forceinline__ uint64_t sum_desc(uint32_t tile) { return smem_desc(tile, TileOf<DP>::BOX, 1024); }

// d = a b^T over the columns of a tile and N rows of another.
template <int DP, int N> __device__ __forceinline__ void mma_scores(bool issue, uint32_t d, uint64_t a, uint64_t b) {
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
        const uint32_t at = (k / 4) * TileOf<DP>::BOX + (k % 4) * 32;
        if (issue)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d), "l"(desc_on(a, at)), "l"(desc_on(b, at)), "r"(IDESC_SCORES<N>), "r"(k ? 1 : 0)
            : "memory");
    }
}

// d (+)= p x: p [128, N] binary16 in TMEM, x N rows of a tile, summed over.
template <int DP, int N> __device__ __forceinline__ void mma_sums(bool issue, uint32_t d, uint32_t p, uint64_t x, bool add) {
#pragma unroll
    for (int k = 0; k < N / 16; ++k)
        if (issue)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
            ::"r"(d), "r"(p + k * 8), "l"(desc_on(x, k * 16 * 128)), "r"(IDESC_SUMS<DP>), "r"(add || k ? 1 : 0)
            : "memory");
}

// 32 columns of this thread's TMEM lane, to be used after tmem_wait on them.
__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// Waits for this thread's loads; ties the registers so that no use is moved before it.
__device__ __forceinline__ void tmem_wait(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
// 16 columns from registers; visible to the tensor core after tmem_st_wait and the fences.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {  // passes over NaN
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float exp2_fast(float x) {  // 2 ulp; 0 below 2^-126
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The bits below n (none for n <= 0, all from 32 on).
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t half2_of(float a, float b) {  // in the order written, as exp2_fast
    uint32_t h;
    asm volatile("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(b), "f"(a));
    return h;
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

// The accumulator truncates: a sum of 8192 numbers of one sign loses 5e-5 of itself, of 131072 9e-4 (an
// output's rounding is 4.9e-4).  Sums over more than DRAIN tiles leave it every DRAIN tiles for binary32 sums
// in memory, by kernels of their own (LONG): the others are 0.5 to 2 % slower with the branches, 32768 tokens
// of 8 heads over 2 take 1.85 -> 1.89 ms, their gradients 6.8 -> 7.0.  A tile's are [D / 4][128 rows][4], so that a
// warp's 16 bytes a lane lie together; only the row's own thread uses them.
constexpr int DRAIN = 64;
// Tiles of keys that a tile of queries meets, at most.
inline int64_t most_key_tiles(const Problem& p) {
    const int64_t all = (static_cast<int64_t>(p.Sk) + TILE - 1) / TILE;
    return p.window ? std::min<int64_t>(all, p.window / TILE + 3 + (p.sinks + TILE - 1) / TILE) : all;
}
// Kept sums of all tiles of queries, [B][Hq][tiles], or null where none meets that many tiles of keys.
inline qsml_status_t get_kept(Workspace* ws, const Problem& p, float** kept) {
    *kept = nullptr;
    if (most_key_tiles(p) <= DRAIN) return QSML_OK;
    void* m = nullptr;
    QSML_TRY_STATUS(ws->get(sizeof(float) * p.B * p.Hq * ((static_cast<size_t>(p.Sq) + TILE - 1) / TILE) * TILE * p.D, &m));
    *kept = static_cast<float*>(m);
    return QSML_OK;
}
// Column c (a multiple of 4) of a row of a tile's kept sums.
__device__ __forceinline__ float* kept_at(float* tile, int row, int c) { return tile + c * TILE + row * 4; }
// 32 columns of a row of sums in TMEM, of which n are in use, with g times what is kept of them (null: nothing).
__device__ __forceinline__ void load_sums(uint32_t taddr, uint32_t (&r)[32], const float* kept, int n, float g) {
    tmem_ld32_start(taddr, r);
    tmem_wait(r);
    if (kept) {
#pragma unroll
        for (int e = 0; e < 32; e += 16) {  // in two batches: all at once cost registers that the steps use
            float4 y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (e + 4 * i < n) y[i] = *reinterpret_cast<const float4*>(kept + (e + 4 * i) * TILE);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (e + 4 * i < n) {
                    const float z[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) r[e + 4 * i + k] = __float_as_uint(fmaf(z[k], g, __uint_as_float(r[e + 4 * i + k])));
                }
        }
    }
}
// A row of sums, D columns from TMEM's, added to g times what is kept of it (first: nothing yet).
template <int DP> __device__ __forceinline__ void keep_sums(uint32_t taddr, float* kept, int D, bool first, float g) {
#pragma unroll
    for (int c = 0; c < DP; c += 32) {
        if (c >= D) break;
        uint32_t r[32];
        load_sums(taddr + c, r, first ? nullptr : kept + c * TILE, D - c, g);
#pragma unroll
        for (int j = 0; j < 32; j += 4)
            if (c + j < D)
                *reinterpret_cast<float4*>(kept + (c + j) * TILE) =
                    make_float4(__uint_as_float(r[j]), __uint_as_float(r[j + 1]), __uint_as_float(r[j + 2]), __uint_as_float(r[j + 3]));
    }
}

// A row of binary32 sums in TMEM, with g times what is kept of it (null: nothing), times f, as binary16 to `to`
// (null: nowhere), D columns.
template <int DP> __device__ __forceinline__ void store_row(uint32_t taddr, float f, __half* to, int D, const float* kept = nullptr, float g = 1.0f) {
#pragma unroll
    for (int c = 0; c < DP; c += 32) {
        if (c >= D) break;
        uint32_t r[32];
        load_sums(taddr + c, r, kept ? kept + c * TILE : nullptr, D - c, g);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (to && c + 8 * j < D) {
                uint4 w;
                uint32_t* h = &w.x;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    h[e] = half2_of(__uint_as_float(r[8 * j + 2 * e]) * f, __uint_as_float(r[8 * j + 2 * e + 1]) * f);
                *reinterpret_cast<uint4*>(to + c + 8 * j) = w;
            }
    }
}
__device__ __forceinline__ void zero_row(__half* to, int D) {
    for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(to + c) = make_uint4(0, 0, 0, 0);
}

}  // namespace attn
}  // namespace qsml
