// Attention and its gradients on the CUDA cores, for binary32 and for what the tensor
// cores' kernels do not take (heads of more than 128 columns, rows off 16 bytes).
//
// A tile of BT queries meets a tile of BT keys, both in shared memory as binary32; 16 x 16
// threads hold RT x RT of its scores (RT = BT / 16) and RT rows x DP / 16 columns of each
// sum.  Products are packed pairs (fma.rn.f32x2).  Forward: one pass over the visible keys
// with each row's running maximum and sum (exp(s - m), the sum and what was summed before
// multiplied by exp(m_old - m) where m grows); nothing of the scores leaves the SM.
// Backward: P = exp(s - lse) again from the kept lse.  dk and dv of a tile of keys are
// summed by one CTA over all queries that see it and all heads of its group, dq of a tile
// of queries by another over its keys: seven products instead of five, no atomics.  Where the tiles
// do not fill the device, each one's steps are split over CTAs whose sums are joined in order.
// Bound by the FFMA pipe and by shared memory, a 16-byte load for 8 multiply-adds; two fifths of that pipe
// at 2048 tokens of 8 heads over 2 of 128 (269 us, 32 TFLOP/s of visible pairs), with two CTAs a SM.
#include <algorithm>
#include <type_traits>

#include "attention.cuh"
#include "packed.cuh"

namespace qsml {
namespace attn {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int DP, int B> struct Shape {
    static constexpr int BT = B;
    static constexpr int RT = BT / 16;   // rows and columns of scores a thread
    static constexpr int CT = DP / 16;   // columns of a sum a thread
    static constexpr int LD = DP + 4;    // floats between rows: 16 lanes' 16-byte loads meet 8 by 8 in no bank
    static constexpr int LP = BT + 4;
    static constexpr int TILE = BT * LD, PROBS = BT * LP;
};

// Rows [r0, r0 + BT) of a head, those in [lo, hi) or below sink, as floats; 0 elsewhere.
template <typename T, int DP, int BT>
__device__ __forceinline__ void load_tile(float* dst, const View& v, int64_t at, int r0, int sink, int lo, int hi, int D, bool vec) {
    using S = Shape<DP, BT>;
    constexpr int V = 16 / sizeof(T);
    const T* p = reinterpret_cast<const T*>(v.p) + at;
    if (vec) {
        // a thread's loads are all on their way before the first is stored
        constexpr int COLS = DP / V, ALL = S::BT * COLS, N = (ALL + kThreads - 1) / kThreads;
        heads::Pack<T, V> x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = threadIdx.x + i * kThreads, c = at % COLS * V, row = r0 + at / COLS;
            const bool in = at < ALL && (row >= lo || row < sink) && row < hi && c < D;
#pragma unroll
            for (int e = 0; e < V; ++e) heads::from_f(0.0f, x[i].v[e]);
            if (in) x[i] = *reinterpret_cast<const heads::Pack<T, V>*>(p + row * v.s + c);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = threadIdx.x + i * kThreads, c = at % COLS * V, r = at / COLS;
            if (ALL % kThreads && at >= ALL) break;
#pragma unroll
            for (int e = 0; e < V; e += 4)
                *reinterpret_cast<float4*>(dst + r * S::LD + c + e) =
                    make_float4(heads::to_f(x[i].v[e]), heads::to_f(x[i].v[e + 1]), heads::to_f(x[i].v[e + 2]), heads::to_f(x[i].v[e + 3]));
        }
    } else {
        for (int i = threadIdx.x; i < S::BT * DP; i += kThreads) {
            const int r = i / DP, c = i % DP, row = r0 + r;
            dst[r * S::LD + c] = (row >= lo || row < sink) && row < hi && c < D ? heads::to_f(p[row * v.s + c]) : 0.0f;
        }
    }
}

// acc[i][j] = sum over columns of a[ty RT + i] b[tx + 16 j].
template <int DP, int BT> __device__ __forceinline__ void dots(int D, const float* a, const float* b, float (&acc)[Shape<DP, BT>::RT][Shape<DP, BT>::RT]) {
    using S = Shape<DP, BT>;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    P2 s[S::RT][S::RT];
#pragma unroll
    for (int i = 0; i < S::RT; ++i)
#pragma unroll
        for (int j = 0; j < S::RT; ++j) s[i][j] = pack(0.0f, 0.0f);
#pragma unroll 4
    for (int c = 0; c < D; c += 4) {
        float4 x[S::RT], y[S::RT];
#pragma unroll
        for (int i = 0; i < S::RT; ++i) x[i] = *reinterpret_cast<const float4*>(a + (ty * S::RT + i) * S::LD + c);
#pragma unroll
        for (int j = 0; j < S::RT; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * S::LD + c);
#pragma unroll
        for (int i = 0; i < S::RT; ++i)
#pragma unroll
            for (int j = 0; j < S::RT; ++j) {
                s[i][j] = fma2(pack(x[i].x, x[i].y), pack(y[j].x, y[j].y), s[i][j]);
                s[i][j] = fma2(pack(x[i].z, x[i].w), pack(y[j].z, y[j].w), s[i][j]);
            }
    }
#pragma unroll
    for (int i = 0; i < S::RT; ++i)
#pragma unroll
        for (int j = 0; j < S::RT; ++j) acc[i][j] = sum2(s[i][j]);
}

// Columns of a thread's sums: 4 tx + 64 n + e, and 2 tx + e of the last 32 where they are half of 64.
template <int DP, int BT> struct Sum {
    static constexpr int FOURS = DP / 64;
    P2 v[Shape<DP, BT>::RT][Shape<DP, BT>::CT / 2];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (auto& r : v)
#pragma unroll
            for (auto& x : r) x = pack(0.0f, 0.0f);
    }
    // += p (rows ty RT + i of [BT][LP]) times x ([BT][LD])
    __device__ __forceinline__ void add(const float* p, const float* x) {
        using S = Shape<DP, BT>;
        const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll 2
        for (int k = 0; k < S::BT; k += 4) {
            float w[S::RT][4];
#pragma unroll
            for (int i = 0; i < S::RT; ++i) *reinterpret_cast<float4*>(w[i]) = *reinterpret_cast<const float4*>(p + (ty * S::RT + i) * S::LP + k);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int n = 0; n < FOURS; ++n) {
                    const float4 y = *reinterpret_cast<const float4*>(x + (k + e) * S::LD + 4 * tx + 64 * n);
#pragma unroll
                    for (int i = 0; i < S::RT; ++i) {
                        v[i][2 * n] = fma2(both(w[i][e]), pack(y.x, y.y), v[i][2 * n]);
                        v[i][2 * n + 1] = fma2(both(w[i][e]), pack(y.z, y.w), v[i][2 * n + 1]);
                    }
                }
            if constexpr (DP % 64 != 0) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 y = *reinterpret_cast<const float2*>(x + (k + e) * S::LD + 2 * tx + 64 * FOURS);
#pragma unroll
                    for (int i = 0; i < S::RT; ++i) v[i][2 * FOURS] = fma2(both(w[i][e]), pack(y.x, y.y), v[i][2 * FOURS]);
                }
            }
        }
    }
    template <typename T> __device__ __forceinline__ void store(int i, T* row, float f, int D) const {
        const int tx = threadIdx.x & 15;
#pragma unroll
        for (int n = 0; n < FOURS; ++n) {
            const float2 a = unpack(v[i][2 * n]), b = unpack(v[i][2 * n + 1]);
            const float y[4] = {a.x * f, a.y * f, b.x * f, b.y * f};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * tx + 64 * n + e < D) heads::from_f(y[e], row[4 * tx + 64 * n + e]);
        }
        if constexpr (DP % 64 != 0) {
            const float2 a = unpack(v[i][2 * FOURS]);
            const int c = 2 * tx + 64 * FOURS;
            if (c < D) heads::from_f(a.x * f, row[c]);
            if (c + 1 < D) heads::from_f(a.y * f, row[c + 1]);
        }
    }
};

__device__ __forceinline__ float row_max(float v) {
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

__device__ __forceinline__ float exp2_fast(float x) {  // 2 ulp; 0 below 2^-126
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Whether every query of [q0, q0 + n), all below nq, sees every key of [k0, k0 + n).
__device__ __forceinline__ bool all_see(const Problem& a, const Seq& s, int q0, int k0, int n) {
    const int pos = q0 + s.nk - s.nq;
    return q0 + n <= s.nq && k0 + n - 1 <= pos && (a.window == 0 || pos + n - 1 - k0 < a.window || k0 + n <= a.sinks);
}

// A CTA's part of a tile's steps, the tile (of queries the last first: with the most keys), head and
// sequence.
struct Where {
    int part, tile, h, b;
    __device__ __forceinline__ Where(int i, int parts, int tiles, int H, bool backwards) {
        part = i % parts;
        i /= parts;
        h = i % H;
        i /= H;
        tile = backwards ? tiles - 1 - i % tiles : i % tiles;
        b = i / tiles;
    }
};
// The steps of a part.
struct Share {
    int lo, hi;
    __device__ __forceinline__ Share(int steps, int parts, int part) {
        const int n = (steps + parts - 1) / parts;
        lo = min(part * n, steps);
        hi = min(lo + n, steps);
    }
};

template <typename T, int DP, int BT>
__global__ void __launch_bounds__(kThreads) k_attention_simt(const __grid_constant__ Problem p, Parts parts, int tiles, bool vec) {
    using S = Shape<DP, BT>;
    extern __shared__ float4 smem[];
    float *sq = reinterpret_cast<float*>(smem), *skv = sq + S::TILE, *sp = skv + S::TILE;
    pdl_begin();
    const Where w(blockIdx.x, parts.parts, tiles, p.Hq, true);
    const Seq seq(p, w.b);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int q0 = w.tile * S::BT, off = seq.nk - seq.nq, hk = w.h / p.G;
    const Keys keys(p, seq.nk, q0 + off, min(q0 + S::BT, seq.nq) - 1 + off);
    const Tiles t(keys, S::BT);
    load_tile<T, DP, BT>(sq, p.q, w.b * p.q.b + w.h * p.q.h, q0, 0, 0, seq.nq, p.D, vec);
    Sum<DP, BT> o;
    o.zero();
    float m[S::RT], l[S::RT];
#pragma unroll
    for (int i = 0; i < S::RT; ++i) m[i] = -INFINITY, l[i] = 0.0f;
    const float c = p.scale * kLog2e;
    const Share steps(q0 < seq.nq ? t.n : 0, parts.parts, w.part);
    for (int n = steps.lo; n < steps.hi; ++n) {
        const int k0 = t.tile(n) * S::BT;
        __syncthreads();
        load_tile<T, DP, BT>(skv, p.k, w.b * p.k.b + hk * p.k.h, k0, 0, 0, seq.nk, p.D, vec);
        __syncthreads();
        float s[S::RT][S::RT];
        dots<DP, BT>(p.D, sq, skv, s);
        const bool whole = all_see(p, seq, q0, k0, S::BT);
#pragma unroll
        for (int i = 0; i < S::RT; ++i) {
            const int pos = q0 + ty * S::RT + i + off;
            float most = -INFINITY;
#pragma unroll
            for (int j = 0; j < S::RT; ++j) {
                s[i][j] = whole || (pos < seq.nk && sees(p, pos, k0 + tx + 16 * j)) ? s[i][j] * c : -INFINITY;
                most = fmaxf(most, s[i][j]);
            }
            const float now = fmaxf(m[i], row_max(most)), ref = now == -INFINITY ? 0.0f : now;
            const float f = exp2_fast(m[i] - ref);
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < S::RT; ++j) {
                const float e = exp2_fast(s[i][j] - ref);
                sum += e;
                sp[(ty * S::RT + i) * S::LP + tx + 16 * j] = e;
            }
            l[i] = fmaf(l[i], f, row_sum(sum));
            m[i] = now;
#pragma unroll
            for (auto& x : o.v[i]) x = mul2(x, both(f));
        }
        __syncthreads();
        // values that no row of the tile sees count for nothing, whatever they are
        load_tile<T, DP, BT>(skv, p.v, w.b * p.v.b + hk * p.v.h, k0, keys.sink, keys.lo, keys.hi, p.D, vec);
        __syncthreads();
        o.add(sp, skv);
    }
#pragma unroll
    for (int i = 0; i < S::RT; ++i) {
        const int q = q0 + ty * S::RT + i;
        if (q >= p.Sq) continue;
        if (parts.parts > 1) {
            const int64_t at = ((static_cast<int64_t>(w.b) * p.Hq + w.h) * p.Sq + q) * parts.parts + w.part;
            o.store(i, parts.sum + at * p.D, 1.0f, p.D);
            if (tx == 0) parts.stat[2 * at] = m[i], parts.stat[2 * at + 1] = l[i];
            continue;
        }
        const bool any = l[i] > 0.0f || isnan(l[i]);
        o.store(i, reinterpret_cast<T*>(p.o.p) + w.b * p.o.b + q * p.o.s + w.h * p.o.h, any ? 1.0f / l[i] : 0.0f, p.D);
        if (p.lse && tx == 0) p.lse[(static_cast<int64_t>(w.b) * p.Hq + w.h) * p.Sq + q] = any ? (m[i] + log2f(l[i])) * kLn2 : -INFINITY;
    }
}

// Shared memory of the gradients' kernels: two fixed tiles, two that come and go, P and dS.
template <int DP, int BT> constexpr size_t grad_smem() { return sizeof(float) * (4 * Shape<DP, BT>::TILE + 2 * Shape<DP, BT>::PROBS + 2 * Shape<DP, BT>::BT); }

// Sums of a gradient in parts: [parts][B][H][S][D] binary32.
struct Sums {
    float* p = nullptr;
    int parts = 1;
    __device__ __forceinline__ float* row(const Problem& a, int part, int b, int h, int H, int i, int S) const {
        return p + (((static_cast<int64_t>(part) * a.B + b) * H + h) * S + i) * a.D;
    }
};

// dk and dv of a tile of keys.
template <typename T, int DP, int BT>
__device__ __forceinline__ void gradients_of_keys(const Problem& p, int cta, const float* delta, const Sums& to_k, const Sums& to_v, int tiles, bool vec) {
    using S = Shape<DP, BT>;
    extern __shared__ float4 smem[];
    float *sk = reinterpret_cast<float*>(smem), *sv = sk + S::TILE, *sq = sv + S::TILE, *sg = sq + S::TILE, *sp = sg + S::TILE,
          *sd = sp + S::PROBS, *sl = sd + S::PROBS, *sdel = sl + S::BT;
    const Where w(cta, to_k.parts, tiles, p.Hk, false);
    const int hk = w.h, b = w.b;
    const Seq seq(p, b);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int k0 = w.tile * S::BT, off = seq.nk - seq.nq;
    load_tile<T, DP, BT>(sk, p.k, b * p.k.b + hk * p.k.h, k0, 0, 0, seq.nk, p.D, vec);
    load_tile<T, DP, BT>(sv, p.v, b * p.v.b + hk * p.v.h, k0, 0, 0, seq.nk, p.D, vec);
    Sum<DP, BT> dk, dv;
    dk.zero();
    dv.zero();
    const Queries qs(p, seq, k0, k0 + S::BT);
    const int t0 = qs.lo / S::BT, per = qs.hi > qs.lo ? (qs.hi + S::BT - 1) / S::BT - t0 : 0;  // tiles of queries a head
    const Share steps(per * p.G, to_k.parts, w.part);
    for (int n = steps.lo; n < steps.hi; ++n) {
        const int h = hk * p.G + n / per, q0 = (t0 + n % per) * S::BT;
        const int64_t stat = (static_cast<int64_t>(b) * p.Hq + h) * p.Sq;
        __syncthreads();
        load_tile<T, DP, BT>(sq, p.q, b * p.q.b + h * p.q.h, q0, 0, 0, seq.nq, p.D, vec);
        load_tile<T, DP, BT>(sg, p.dout, b * p.dout.b + h * p.dout.h, q0, 0, 0, seq.nq, p.D, vec);
        if (threadIdx.x < S::BT) {
            const int q = q0 + threadIdx.x;
            sl[threadIdx.x] = q < seq.nq ? p.lse[stat + q] : 0.0f;
            sdel[threadIdx.x] = q < seq.nq ? delta[stat + q] : 0.0f;
        }
        __syncthreads();
        float s[S::RT][S::RT], d[S::RT][S::RT];
        dots<DP, BT>(p.D, sk, sq, s);
        dots<DP, BT>(p.D, sv, sg, d);
        const bool whole = all_see(p, seq, q0, k0, S::BT);
#pragma unroll
        for (int i = 0; i < S::RT; ++i)
#pragma unroll
            for (int j = 0; j < S::RT; ++j) {
                const int key = k0 + ty * S::RT + i, q = tx + 16 * j;
                const bool seen = whole || (q0 + q < seq.nq && sees(p, q0 + q + off, key));
                const float e = seen ? exp2_fast((s[i][j] * p.scale - sl[q]) * kLog2e) : 0.0f;
                sp[(ty * S::RT + i) * S::LP + q] = e;
                sd[(ty * S::RT + i) * S::LP + q] = seen && !sees_one(p, q0 + q + off) ? e * (d[i][j] - sdel[q]) : 0.0f;
            }
        __syncthreads();
        dv.add(sp, sg);
        dk.add(sd, sq);
    }
#pragma unroll
    for (int i = 0; i < S::RT; ++i) {
        const int k = k0 + ty * S::RT + i;
        if (k >= p.Sk) continue;
        if (to_k.parts > 1) {
            if (p.dk.p) dk.store(i, to_k.row(p, w.part, b, hk, p.Hk, k, p.Sk), p.scale, p.D);
            if (p.dv.p) dv.store(i, to_v.row(p, w.part, b, hk, p.Hk, k, p.Sk), 1.0f, p.D);
            continue;
        }
        if (p.dk.p) dk.store(i, reinterpret_cast<T*>(p.dk.p) + b * p.dk.b + k * p.dk.s + hk * p.dk.h, p.scale, p.D);
        if (p.dv.p) dv.store(i, reinterpret_cast<T*>(p.dv.p) + b * p.dv.b + k * p.dv.s + hk * p.dv.h, 1.0f, p.D);
    }
}

// dq of a tile of queries.
template <typename T, int DP, int BT>
__device__ __forceinline__ void gradients_of_queries(const Problem& p, int cta, const float* delta, const Sums& to, int tiles, bool vec) {
    using S = Shape<DP, BT>;
    extern __shared__ float4 smem[];
    float *sq = reinterpret_cast<float*>(smem), *sg = sq + S::TILE, *sk = sg + S::TILE, *sv = sk + S::TILE, *sd = sv + S::TILE;
    const Where w(cta, to.parts, tiles, p.Hq, true);
    const Seq seq(p, w.b);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int q0 = w.tile * S::BT, off = seq.nk - seq.nq, hk = w.h / p.G;
    const Keys keys(p, seq.nk, q0 + off, min(q0 + S::BT, seq.nq) - 1 + off);
    const Tiles t(keys, S::BT);
    load_tile<T, DP, BT>(sq, p.q, w.b * p.q.b + w.h * p.q.h, q0, 0, 0, seq.nq, p.D, vec);
    load_tile<T, DP, BT>(sg, p.dout, w.b * p.dout.b + w.h * p.dout.h, q0, 0, 0, seq.nq, p.D, vec);
    Sum<DP, BT> dq;
    dq.zero();
    const int64_t stat = (static_cast<int64_t>(w.b) * p.Hq + w.h) * p.Sq;
    float lse[S::RT], del[S::RT];
#pragma unroll
    for (int i = 0; i < S::RT; ++i) {
        const int q = q0 + ty * S::RT + i;
        lse[i] = q < seq.nq ? p.lse[stat + q] : 0.0f;
        del[i] = q < seq.nq ? delta[stat + q] : 0.0f;
    }
    const Share steps(q0 < seq.nq ? t.n : 0, to.parts, w.part);
    for (int n = steps.lo; n < steps.hi; ++n) {
        const int k0 = t.tile(n) * S::BT;
        __syncthreads();
        load_tile<T, DP, BT>(sk, p.k, w.b * p.k.b + hk * p.k.h, k0, keys.sink, keys.lo, keys.hi, p.D, vec);
        load_tile<T, DP, BT>(sv, p.v, w.b * p.v.b + hk * p.v.h, k0, keys.sink, keys.lo, keys.hi, p.D, vec);
        __syncthreads();
        float s[S::RT][S::RT], d[S::RT][S::RT];
        dots<DP, BT>(p.D, sq, sk, s);
        dots<DP, BT>(p.D, sg, sv, d);
        const bool whole = all_see(p, seq, q0, k0, S::BT);
#pragma unroll
        for (int i = 0; i < S::RT; ++i)
#pragma unroll
            for (int j = 0; j < S::RT; ++j) {
                const int q = q0 + ty * S::RT + i;
                const bool seen = whole || (q < seq.nq && sees(p, q + off, k0 + tx + 16 * j));
                const float e = seen ? exp2_fast((s[i][j] * p.scale - lse[i]) * kLog2e) : 0.0f;
                sd[(ty * S::RT + i) * S::LP + tx + 16 * j] = seen && !sees_one(p, q + off) ? e * (d[i][j] - del[i]) : 0.0f;
            }
        __syncthreads();
        dq.add(sd, sk);
    }
#pragma unroll
    for (int i = 0; i < S::RT; ++i) {
        const int q = q0 + ty * S::RT + i;
        if (q >= p.Sq) continue;
        if (to.parts > 1)
            dq.store(i, to.row(p, w.part, w.b, w.h, p.Hq, q, p.Sq), p.scale, p.D);
        else
            dq.store(i, reinterpret_cast<T*>(p.dq.p) + w.b * p.dq.b + q * p.dq.s + w.h * p.dq.h, p.scale, p.D);
    }
}

// The first key_ctas CTAs have keys, the others queries.
template <typename T, int DP, int BT>
__global__ void __launch_bounds__(kThreads)
    k_attention_bwd_simt(const __grid_constant__ Problem p, const float* delta, Sums to_q, Sums to_k, Sums to_v, int key_ctas, int tq, int tk, bool vec) {
    pdl_begin();
    if (static_cast<int>(blockIdx.x) < key_ctas)
        gradients_of_keys<T, DP, BT>(p, blockIdx.x, delta, to_k, to_v, tk, vec);
    else
        gradients_of_queries<T, DP, BT>(p, blockIdx.x - key_ctas, delta, to_q, tq, vec);
}

// The gradients of which there are parts (dq, dk, dv by blockIdx.y): their sums, added in order.
template <typename T> __global__ void __launch_bounds__(256) k_attention_sum(const __grid_constant__ Problem p, Sums to_q, Sums to_k, Sums to_v) {
    pdl_begin();
    const int which = blockIdx.y, H = which ? p.Hk : p.Hq, S = which ? p.Sk : p.Sq;
    const Sums& from = which == 0 ? to_q : which == 1 ? to_k : to_v;
    const View& out = which == 0 ? p.dq : which == 1 ? p.dk : p.dv;
    if (!out.p || from.parts == 1) return;
    const int64_t n = static_cast<int64_t>(p.B) * H * S * p.D;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
        float v = 0.0f;
#pragma unroll 4
        for (int k = 0; k < from.parts; ++k) v += from.p[k * n + i];
        const int c = static_cast<int>(i % p.D);
        const int64_t row = i / p.D;
        const int s = static_cast<int>(row % S), h = static_cast<int>(row / S % H), b = static_cast<int>(row / S / H);
        heads::from_f(v, reinterpret_cast<T*>(out.p)[b * out.b + s * out.s + h * out.h + c]);
    }
}

// Whether all rows read can be read in 16 bytes.
bool whole(const Problem& p, bool backward) {
    const int64_t es = p.f16 ? 2 : 4;
    bool ok = p.D * es % 16 == 0 && heads::rows_on(p.q, es, 16) && heads::rows_on(p.k, es, 16) && heads::rows_on(p.v, es, 16);
    return ok && (!backward || heads::rows_on(p.dout, es, 16));
}

// Parts of each of `ctas` tiles of at most `steps` steps: enough for four CTAs a SM.  2048 tokens of 8
// heads over 2 with 128 columns, binary32: gradients 2535 -> 918 us, 3 x 200 of 6 over 3: 193 -> 72.
int64_t parts_of(Context* ctx, int64_t ctas, int64_t steps) {
    const int64_t want = (4 * static_cast<int64_t>(ctx->num_sms) + ctas - 1) / std::max<int64_t>(ctas, 1);
    return std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, 16), steps));
}

template <typename K, typename... A>
qsml_status_t launch(Context* ctx, K kernel, const char* name, size_t smem, int64_t ctas, A... args) {
    if (ctas > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "qsml_attention: dimensions too large");
    QSML_TRY_STATUS(check_cuda(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)), name));
    const cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), smem, ctx->stream, args...);
    if (e != cudaSuccess) return check_cuda(ctx, e, name);
    return after_launch(ctx, name);
}

// f(width, tile) with constants: tiles of 64, or of 32 for more than 128 columns and where there are few
// steps of 64 (up to SMALL a SM), which take four times as long: 64 tokens of one head of 128, binary32,
// gradients 41 -> 26 us.  With 24 for SMALL 2 x 777 tokens take 282 us instead of 225.
template <typename F> qsml_status_t by_shape(Context* ctx, const Problem& p, int64_t heads, F&& f) {
    constexpr int64_t SMALL = 8;
    const int64_t tq = (p.Sq + 63) / 64, tk = std::min<int64_t>((p.Sk + 63) / 64, p.window ? (static_cast<int64_t>(p.window) + p.sinks) / 64 + 2 : p.Sk);
    const bool small = tq * tk * heads * p.B <= SMALL * ctx->num_sms;
    return by_width(p.D, [&](auto width) {
        if constexpr (decltype(width)::value <= 128)
            if (!small) return f(width, std::integral_constant<int, 64>());
        return f(width, std::integral_constant<int, 32>());
    });
}

template <typename T> qsml_status_t forward(Context* ctx, const Problem& p) {
    return by_shape(ctx, p, p.Hq, [&](auto width, auto tile) {
        constexpr int DP = decltype(width)::value, BT = decltype(tile)::value;
        using S = Shape<DP, BT>;
        const int tiles = (p.Sq + S::BT - 1) / S::BT;
        const int64_t ctas = static_cast<int64_t>(tiles) * p.Hq * p.B;
        Workspace ws(ctx);
        Parts parts;
        QSML_TRY_STATUS(get_parts(ctx, &ws, p, parts_of(ctx, ctas, (p.Sk + S::BT - 1) / S::BT), &parts));
        QSML_TRY_STATUS(launch(ctx, k_attention_simt<T, DP, BT>, "k_attention_simt", sizeof(float) * (2 * S::TILE + S::PROBS), ctas * parts.parts, p, parts,
                               tiles, whole(p, false)));
        return join_parts(ctx, p, parts);
    });
}

template <typename T> qsml_status_t backward(Context* ctx, const Problem& p, const float* delta) {
    return by_shape(ctx, p, p.Hq, [&](auto width, auto tile) {
        constexpr int DP = decltype(width)::value, BT = decltype(tile)::value;
        using S = Shape<DP, BT>;
        const bool vec = whole(p, true);
        const int tq = (p.Sq + S::BT - 1) / S::BT, tk = (p.Sk + S::BT - 1) / S::BT;
        Workspace ws(ctx);
        auto sums = [&](int64_t parts, int H, int Sn, Sums* out) {
            out->parts = static_cast<int>(parts);
            void* m = nullptr;
            if (parts > 1) QSML_TRY_STATUS(ws.get(sizeof(float) * parts * p.B * H * Sn * p.D, &m));
            out->p = static_cast<float*>(m);
            return static_cast<qsml_status_t>(QSML_OK);
        };
        const bool keys = p.dk.p || p.dv.p, queries = p.dq.p != nullptr;
        const int64_t kc = keys ? static_cast<int64_t>(tk) * p.Hk * p.B : 0, qc = queries ? static_cast<int64_t>(tq) * p.Hq * p.B : 0;
        const int64_t kparts = keys ? parts_of(ctx, kc, static_cast<int64_t>(tq) * p.G) : 1, qparts = queries ? parts_of(ctx, qc, tk) : 1;
        Sums to_q, to_k, to_v;
        QSML_TRY_STATUS(sums(qparts, p.Hq, p.Sq, &to_q));
        QSML_TRY_STATUS(sums(kparts, p.Hk, p.Sk, &to_k));
        QSML_TRY_STATUS(sums(kparts, p.Hk, p.Sk, &to_v));
        if (kc * kparts > INT32_MAX) return set_error(ctx, QSML_E_UNSUPPORTED, "qsml_attention_backward: dimensions too large");
        QSML_TRY_STATUS((launch(ctx, k_attention_bwd_simt<T, DP, BT>, "k_attention_bwd_simt", grad_smem<DP, BT>(), kc * kparts + qc * qparts, p, delta, to_q,
                                to_k, to_v, static_cast<int>(kc * kparts), tq, tk, vec)));
        if (kparts > 1 || qparts > 1) {
            const int64_t most = std::max(static_cast<int64_t>(p.Hq) * p.Sq, static_cast<int64_t>(p.Hk) * p.Sk) * p.B * p.D;
            const dim3 grid(static_cast<unsigned>(std::min<int64_t>((most + 255) / 256, 8 * ctx->num_sms)), 3);
            const cudaError_t e = launch_pdl(k_attention_sum<T>, grid, dim3(256), 0, ctx->stream, p, to_q, to_k, to_v);
            if (e != cudaSuccess) return check_cuda(ctx, e, "k_attention_sum");
            QSML_TRY_STATUS(after_launch(ctx, "k_attention_sum"));
        }
        return static_cast<qsml_status_t>(QSML_OK);
    });
}

}  // namespace

qsml_status_t forward_simt(Context* ctx, const Problem& p) { return p.f16 ? forward<__half>(ctx, p) : forward<float>(ctx, p); }
qsml_status_t backward_simt(Context* ctx, const Problem& p, const float* delta) {
    return p.f16 ? backward<__half>(ctx, p, delta) : backward<float>(ctx, p, delta);
}

}  // namespace attn
}  // namespace qsml
