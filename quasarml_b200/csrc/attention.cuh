// A problem of qsml_attention or its backward pass, and which keys a query sees.
#pragma once

#include "heads.cuh"

namespace qsml {
namespace attn {

using heads::View;

struct Problem {
    View q, k, v, o, dout;       // o: written by the forward pass, read by the backward
    View dq, dk, dv;             // p null: not wanted
    float* lse = nullptr;        // [B, Hq, Sq], or null
    const int *nq = nullptr, *nk = nullptr;  // lengths of the sequences, or null
    int64_t nq_step = 0, nk_step = 0;
    int B = 0, Hq = 0, Hk = 0, G = 1, D = 0, Sq = 0, Sk = 0;
    int window = 0, sinks = 0;   // window 0: all
    float scale = 1.0f;
    bool f16 = false;
};

// Queries and keys of sequence b.
struct Seq {
    int nq, nk;
    __device__ __forceinline__ Seq(const Problem& p, int b) {
        nq = p.nq ? min(max(p.nq[b * p.nq_step], 0), p.Sq) : p.Sq;
        nk = p.nk ? min(max(p.nk[b * p.nk_step], 0), p.Sk) : p.Sk;
    }
};

// Whether the query at position p (below nk) sees key j.
__device__ __forceinline__ bool sees(const Problem& a, int p, int j) {
    return j <= p && (a.window == 0 || p - j < a.window || j < a.sinks);
}

// Whether the query at position p sees one key alone: its weight is 1 whatever the score, and its dS is 0,
// which P (dP - delta) is only but for their roundings.
__device__ __forceinline__ bool sees_one(const Problem& a, int p) { return p == 0 || (a.window == 1 && a.sinks == 0); }

// The keys that some query of positions [p0, p1] sees: the sinks [0, sink) and [lo, hi),
// with sink <= lo.
struct Keys {
    int sink, lo, hi;
    __device__ __forceinline__ Keys(const Problem& a, int nk, int p0, int p1) {
        hi = max(min(nk, p1 + 1), 0);
        lo = a.window && p0 >= a.window ? p0 - a.window + 1 : 0;
        lo = min(lo, hi);
        sink = min(a.sinks, lo);
    }
    __device__ __forceinline__ int count() const { return sink + hi - lo; }
    // the n-th of them
    __device__ __forceinline__ int key(int n) const { return n < sink ? n : lo + n - sink; }
};

// The tiles of KT keys that hold them, in ascending order.
struct Tiles {
    int first, from, n;  // [0, first) and [from, from + n - first)
    __device__ __forceinline__ Tiles(const Keys& k, int KT) {
        first = (k.sink + KT - 1) / KT;
        from = max(k.lo / KT, first);
        const int end = (k.hi + KT - 1) / KT;
        n = k.hi > k.lo ? first + max(end - from, 0) : first;
    }
    __device__ __forceinline__ int tile(int i) const { return i < first ? i : from + i - first; }
};

// The queries of a sequence that may see a key of [k0, k1): [lo, hi).
struct Queries {
    int lo, hi;
    __device__ __forceinline__ Queries(const Problem& a, const Seq& s, int k0, int k1) {
        const int off = s.nk - s.nq;  // position of query 0
        lo = max(k0 - off, 0);
        hi = s.nq;
        if (a.window && k0 >= a.sinks) {
            const int64_t last = static_cast<int64_t>(min(k1, s.nk)) - 1 + a.window - off;  // first that sees none
            hi = static_cast<int>(last < hi ? max(last, static_cast<int64_t>(0)) : hi);
        }
        if (k0 >= s.nk) hi = lo;
    }
};

// o and lse by CUDA cores (attention_simt.cu); any sizes and alignment.
qsml_status_t forward_simt(Context* ctx, const Problem& p);
// dq, dk, dv by CUDA cores.  delta [B, Hq, Sq]: each row's sum of dout * o.
qsml_status_t backward_simt(Context* ctx, const Problem& p, const float* delta);
// o and lse by the tensor cores (attention_tc.cu), where tc_takes: F16, rows on 16 bytes, up to 128 columns.
bool tc_takes(const Problem& p);
qsml_status_t forward_tc(Context* ctx, const Problem& p);
// dq, dk, dv by the tensor cores (attention_tc_bwd.cu).
bool tc_takes_backward(const Problem& p);
qsml_status_t backward_tc(Context* ctx, const Problem& p);
// A row's keys in parts, row = (b Hq + h) Sq + query: each part's sum, maximum (base 2, scaled) and norm.
struct Parts {
    float* sum = nullptr;   // [rows][parts][D], not divided by l; on 16 bytes
    float* stat = nullptr;  // [rows][parts][2]: m, l, read as pairs; on 16 bytes
    int parts = 1;
};
// Room for them in ws, where there is more than one.
qsml_status_t get_parts(Context* ctx, Workspace* ws, const Problem& p, int64_t parts, Parts* out);
// o and lse from the parts, in their order (attention_few.cu).
qsml_status_t join_parts(Context* ctx, const Problem& p, const Parts& parts);
// Parts of a row's keys for `groups` CTAs, of which a SM holds `resident`, each part of `least` keys or more and,
// as far as that many parts can be joined, of `longest` or less.
int64_t few_parts(Context* ctx, const Problem& p, int64_t groups, int resident, int least, int64_t longest);
// Few queries over many keys: binary16 on the tensor cores, where few_tc_takes (attention_few_tc.cu).
bool few_tc_takes(const Problem& p);
qsml_status_t forward_few_tc(Context* ctx, const Problem& p);
// And by CUDA cores (attention_few.cu).
bool few_queries(const Problem& p);
qsml_status_t forward_few(Context* ctx, const Problem& p);

// Calls f with the least of the widths that hold D columns as a constant.
template <typename F> qsml_status_t by_width(int D, F&& f) {
    if (D <= 64) return f(std::integral_constant<int, 64>());
    if (D <= 96) return f(std::integral_constant<int, 96>());
    if (D <= 128) return f(std::integral_constant<int, 128>());
    return f(std::integral_constant<int, 256>());
}

}  // namespace attn
}  // namespace qsml
