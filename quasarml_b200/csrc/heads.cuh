// Tensors of attention heads, [tokens, heads, columns] or [sequences, tokens, heads,
// columns] with any strides but the last, as the rotary and attention kernels take them.
#pragma once

#include "workspace.cuh"

namespace qsml {
namespace heads {

// Elements between sequences, tokens and heads; the columns of a head lie side by side.
struct View {
    char* p = nullptr;
    int64_t b = 0, s = 0, h = 0;
};

struct Dims {
    int64_t B = 1, S = 0, H = 0, D = 0;
};

struct Named {
    const qsml_tdesc* d;
    const char* name;
};

inline qsml_status_t fail(Context* ctx, qsml_status_t st, const char* op, const std::string& what) {
    return set_error(ctx, st, std::string(op) + ": " + what);
}

// t as heads: its sizes and, where it has elements, its strides.  An output may not
// address an element twice.
inline qsml_status_t view_of(Context* ctx, const char* op, Named t, bool output, Dims* dims, View* view) {
    const qsml_tdesc* d = t.d;
    if (d->ndim != 3 && d->ndim != 4)
        return fail(ctx, QSML_E_SHAPE, op, std::string(t.name) + " must be [tokens, heads, columns] or [sequences, tokens, heads, columns]");
    const int o = d->ndim - 3;
    *dims = Dims{o ? d->shape[0] : 1, d->shape[o], d->shape[o + 1], d->shape[o + 2]};
    *view = View{static_cast<char*>(d->data), o ? d->stride[0] : 0, d->stride[o], d->stride[o + 1]};
    if (dims->B == 1) view->b = 0;
    if (dims->S == 1) view->s = 0;
    if (dims->H == 1) view->h = 0;
    if (numel(d) == 0) return QSML_OK;
    if (dims->D > 1 && d->stride[o + 2] != 1)
        return fail(ctx, QSML_E_UNSUPPORTED, op, std::string(t.name) + " needs unit stride in its last dim (materialise with qsml_gather)");
    if (output) {  // from the smallest stride up, each beyond what lies below it
        int64_t n[3] = {dims->H, dims->S, dims->B}, s[3] = {view->h, view->s, view->b}, extent = dims->D;
        for (int k = 0; k < 3; ++k) {
            int least = -1;
            for (int i = 0; i < 3; ++i)
                if (n[i] > 1 && (least < 0 || s[i] < s[least])) least = i;
            if (least < 0) break;
            if (s[least] < extent)
                return fail(ctx, QSML_E_UNSUPPORTED, op, std::string(t.name) + " addresses an element twice");
            extent += (n[least] - 1) * s[least];
            n[least] = 1;
        }
    }
    return QSML_OK;
}

inline bool same_view(const qsml_tdesc* a, const qsml_tdesc* b) {
    if (a->data != b->data || a->dtype != b->dtype || a->ndim != b->ndim) return false;
    for (int i = 0; i < a->ndim; ++i)
        if (a->shape[i] != b->shape[i] || (a->shape[i] > 1 && a->stride[i] != b->stride[i])) return false;
    return true;
}

// Whether two tensors share bytes.  Heads of one projection ([tokens, all heads, columns]
// sliced by head) have spans that meet though no element does: with one token stride, which
// a sequence's is a whole number of, they are apart if their parts of a token are.
inline bool meet(const qsml_tdesc* a, const qsml_tdesc* b) {
    if (!views_meet(a, b)) return false;
    if (a->ndim < 3 || a->ndim > 4 || b->ndim < 3 || b->ndim > 4 || a->dtype != b->dtype) return true;
    const int64_t es = dtype_size(a->dtype);
    struct Part {
        int64_t step, extent;
        bool ok;
    };
    auto part = [](const qsml_tdesc* d) {
        const int o = d->ndim - 3;
        const int64_t S = d->shape[o], H = d->shape[o + 1], D = d->shape[o + 2], h = d->stride[o + 1];
        const int64_t B = o ? d->shape[0] : 1, bs = o ? d->stride[0] : 0;
        const int64_t step = S > 1 ? d->stride[o] : bs;
        Part p{step, (H - 1) * h + D, step > 0 && h >= 0 && (D == 1 || d->stride[o + 2] == 1)};
        if (p.ok && S > 1 && B > 1) p.ok = bs % step == 0;
        p.ok = p.ok && p.extent <= step;
        return p;
    };
    const Part x = part(a), y = part(b);
    if (!x.ok || !y.ok || x.step != y.step) return true;
    const int64_t bytes = static_cast<const char*>(b->data) - static_cast<const char*>(a->data);
    if (bytes % es) return true;
    int64_t delta = bytes / es % x.step;
    if (delta < 0) delta += x.step;
    return !(delta >= x.extent && delta + y.extent <= x.step);
}

// No output may meet an input or another output; out[i] may be in[i] itself for i < inplace.
inline qsml_status_t check_overlap(Context* ctx, const char* op, const Named* in, int ni, const Named* out, int no, int inplace = 0) {
    for (int o = 0; o < no; ++o) {
        if (!out[o].d) continue;
        for (int i = 0; i < ni; ++i) {
            if (!in[i].d || (i == o && i < inplace && same_view(in[i].d, out[o].d))) continue;
            if (meet(out[o].d, in[i].d))
                return fail(ctx, QSML_E_INVALID, op, std::string(out[o].name) + " overlaps " + in[i].name);
        }
        for (int i = 0; i < o; ++i)
            if (out[i].d && meet(out[o].d, out[i].d))
                return fail(ctx, QSML_E_INVALID, op, std::string(out[o].name) + " overlaps " + out[i].name);
    }
    return QSML_OK;
}

// Whether every row of the view starts on a multiple of `bytes`.
inline bool rows_on(const View& v, int64_t es, int64_t bytes) {
    return reinterpret_cast<uintptr_t>(v.p) % bytes == 0 && v.b * es % bytes == 0 && v.s * es % bytes == 0 && v.h * es % bytes == 0;
}

template <typename T, int N> struct alignas(N * sizeof(T)) Pack {
    T v[N];
};
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f(float v, __half& o) { o = __float2half_rn(v); }

}  // namespace heads
}  // namespace qsml
